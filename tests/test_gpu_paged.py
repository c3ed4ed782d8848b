"""The paged cache's operators against a plain implementation in 64 bits.

Tolerances.  ``u`` is half a step of the result's type (bf16 2^-8, float16 2^-11, relative; float16 below 2^-14: 2^-25 absolute).
    append  the norm's sum of 128 squares and the rotation in 32 bits: at most 140 steps of 2^-24 on |a| + |b|, the pair a rotation
            mixes; one rounding.
    decode  queries and weights enter the products as sums of two 16-bit values: 2^-16 relative in bf16 (2^-8 of a residue that is 2^-8).
            A score is off by at most d = (2^-16 + 130 * 2^-23) * scale * sum |q k| (128 products added in 32 bits), a weight by
            the factor e^(2 d) against the others; sums over n rows of weights times values A = sum p |v| / sum p, 32 bits: (n + 130) * 2^-23.
    attend  tcgen05: scores without the 2^-16, weights rounded once to the pages' type (u), a quarter of them by a polynomial with
            7.5e-5, its relative error, on both sides of the quotient; float16 weights below 2^-14 lose 2^-25 each of a largest
            weight of 1 at least.
"""
import math

import pytest
import torch

from gpu_util import assert_close_bf16

pytestmark = pytest.mark.gpu

D, SCALE, EPS = 128, 0.12, 2.0 ** -23
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype)


def _tables(n=4096):
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return a.cos().float(), a.sin().float()


def _norm(x):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()


def _rotate(x, pos, cos, sin):
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def _mixed(x):
    a = x[..., :64].abs() + x[..., 64:].abs()
    return torch.cat([a, a], -1)


def _check(got, ref, tol, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), f"{what}: {over.max().item():.3g} over the tolerance, off by {(got - ref).abs().max().item():.3g}"


def _store_tol(ref, mixed, dtype):
    tol = HALF[dtype] * ref.abs() + 140 * 2.0 ** -24 * mixed * (1 + HALF[dtype])
    return tol + (2.0 ** -25 if dtype == torch.float16 else 0.0)


class Pool:
    """Pages in a shuffled order on the CPU, every row that nobody wrote poisoned; ``gpu()`` puts it on the device."""

    def __init__(self, lens, new, H, page, dtype, seed, spare=3, window=None, extra_entries=1, unit=True, strided=False):
        g = _gen(seed)
        self.H, self.page, self.dtype = H, page, dtype
        ends = [max(n, 0) + m for n, m in zip(lens, new)]
        need = [-(-e // page) for e in ends]
        order = torch.randperm(sum(need) + spare, generator=g).tolist()
        self.table = torch.full((len(lens), max(need + [1]) + extra_entries), -1, dtype=torch.int32)
        shape = (len(order), H, page, D)
        self.k, self.v = torch.full(shape, float("nan"), dtype=dtype), torch.full(shape, float("inf"), dtype=dtype)
        for b, n in enumerate(need):
            first = 0 if window is None else max(0, max(lens[b], 0) - window + 1) // page
            for i in range(n):
                pg = order.pop()
                if i < first:                                        # behind the window: given back, maybe somebody else's
                    continue
                self.table[b, i] = pg
                rows = min(page, max(lens[b], 0) - i * page)
                if rows > 0:
                    for pool in (self.k, self.v):
                        x = torch.randn(H, rows, D, generator=g)
                        if unit:
                            x = x / x.square().mean(-1, keepdim=True).sqrt()
                        pool[pg, :, :rows] = x.to(dtype)
                if window is not None:                               # rows that the first query does not see any more
                    dead = min(max(0, max(lens[b], 0) - window + 1) - i * page, page)
                    if dead > 0:
                        self.k[pg, :, :dead], self.v[pg, :, :dead] = float("inf"), float("nan")
        self.strided = strided

    def gpu(self):
        if not self.strided:
            return self.k.cuda(), self.v.cuda(), self.table.cuda()
        out = []                                                     # pages of a larger pool: gaps between rows, heads and pages
        for pool in (self.k, self.v):
            big = torch.full((pool.shape[0], self.H + 1, self.page, D + 16), 7.0, dtype=self.dtype, device="cuda")
            big[:, :self.H, :, 8:8 + D] = pool.cuda()
            out.append(big[:, :self.H, :, 8:8 + D])
        wide = torch.full((self.table.shape[0], self.table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device="cuda")
        wide[:, :self.table.shape[1]] = self.table.cuda()
        return out[0], out[1], wide[:, :self.table.shape[1]]

    def row(self, pool, b, pos):
        return pool[self.table[b, pos // self.page].item(), :, pos % self.page]

    def rows(self, pool, b, lo, hi):
        """``[H, hi - lo, D]`` in 64 bits."""
        return torch.stack([self.row(pool, b, p) for p in range(lo, hi)], 1).double() if hi > lo else torch.zeros(self.H, 0, D, dtype=torch.float64)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _status(expect=0):
    from daisy_b200 import _lib, ops
    dev = torch.device("cuda", 0)
    if expect == 0:
        ops.check_device_status(dev)
    else:
        with pytest.raises(_lib.DaisyB200Error) as e:
            ops.check_device_status(dev)
        assert e.value.code == expect


def _same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


# ---------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("starts,counts,Hq,H,page", [
    ([0], [1], 2, 2, 16), ([5], [1], 6, 3, 64), ([15, 16, 17], [1, 1, 1], 3, 3, 16), ([0, 7, 100], [40, 40, 40], 4, 1, 32),
    ([3, 0, 250, 31, 9], [0, 70, 5, 0, 1], 4, 2, 64), ([0, 600], [257, 300], 8, 8, 128), ([0, 1000, 3], [33, 1, 600], 2, 2, 256),
    ([9 * b % 40 for b in range(40)], [5 * b % 7 for b in range(40)], 2, 1, 16), ([13 * b % 60 for b in range(1500)], [7 * b % 4 for b in range(1500)], 1, 1, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("strided", [False, True])
def test_append(starts, counts, Hq, H, page, dtype, strided):
    from daisy_b200 import ops
    packed = len(set(counts)) > 1 or strided
    n, N = len(starts), sum(counts)
    pool = Pool(starts, counts, H, page, dtype, seed=N, strided=strided)
    g = _gen(N + 1)
    qkv = _randn(g, N, Hq + 2 * H, D) * 3
    cos, sin = _tables()
    k_pages, v_pages, table = pool.gpu()
    before = k_pages.clone(), v_pages.clone()
    x = qkv.cuda().unflatten(0, (1, N) if packed else (n, counts[0]))
    cu = _ints([sum(counts[:i]) for i in range(n + 1)]) if packed else None
    q_out = ops.paged_append(x[:, :, Hq:Hq + H], x[:, :, Hq + H:], k_pages, v_pages, table, _ints(starts), cos.cuda(), sin.cuda(), cu_seqlens=cu, q=x[:, :, :Hq], eps=EPS)
    _status()
    assert q_out.dtype == dtype and q_out.shape == (*x.shape[:2], Hq, D)
    pos = torch.tensor([s + i for s, c in zip(starts, counts) for i in range(c)])
    seq = [b for b, c in enumerate(counts) for _ in range(c)]
    qn, kn, vn = (_norm(t) for t in qkv.split([Hq, H, H], 1))
    _check(q_out.flatten(0, 1), _rotate(qn, pos, cos, sin), _store_tol(_rotate(qn, pos, cos, sin), _mixed(qn), dtype), "q")
    kr = _rotate(kn, pos, cos, sin)
    kc, vc = k_pages.cpu(), v_pages.cpu()
    got_k = torch.stack([pool.row(kc, b, p) for b, p in zip(seq, pos.tolist())])
    got_v = torch.stack([pool.row(vc, b, p) for b, p in zip(seq, pos.tolist())])
    _check(got_k, kr, _store_tol(kr, _mixed(kn), dtype), "k")
    _check(got_v, vn, _store_tol(vn, vn.abs(), dtype), "v")
    for i, (b, p) in enumerate(zip(seq, pos.tolist())):              # everything else as it was
        pg, r = pool.table[b, p // page].item(), p % page
        before[0][pg, :, r], before[1][pg, :, r] = k_pages[pg, :, r], v_pages[pg, :, r]
    assert _same_bits(before[0], k_pages) and _same_bits(before[1], v_pages)


def test_append_without_queries_idle_sequences_and_tokens_of_nobody():
    from daisy_b200 import ops
    starts, counts, H = [4, -1, 20], [3, 5, 6], 2
    pool = Pool([4, 0, 20], counts, H, 16, torch.bfloat16, seed=3)
    N, tail = sum(counts), 4
    kv = (_randn(_gen(4), 1, N + tail, 2 * H, D)).cuda()
    k_pages, v_pages, table = pool.gpu()
    before = k_pages.clone()
    cos, sin = _tables()
    cu = [0, 3, 8, 14]
    assert ops.paged_append(kv[:, :, :H], kv[:, :, H:], k_pages, v_pages, table, _ints(starts), None, None, cu_seqlens=_ints(cu), flags=0) is None
    _status()
    for b, (s, c) in enumerate(zip(starts, counts)):
        for i in range(c):
            at = (pool.table[b, (max(s, 0) + i) // 16].item(), (max(s, 0) + i) % 16)
            if s < 0:
                assert torch.isnan(k_pages[at[0], :, at[1]]).all()
            else:                                                    # no norm, no rotation: the values themselves
                assert torch.equal(k_pages[at[0], :, at[1]], kv[0, cu[b] + i, :H]) and torch.equal(v_pages[at[0], :, at[1]], kv[0, cu[b] + i, H:])
                before[at[0], :, at[1]] = k_pages[at[0], :, at[1]]
    assert _same_bits(before, k_pages)
    # a first offset above zero: the tokens in front belong to nobody either
    k2, v2, _ = pool.gpu()
    ops.paged_append(kv[:, :, :H], kv[:, :, H:], k2, v2, table, _ints([4, 0, 20]), None, None, cu_seqlens=_ints([2, 3, 3, 5]), flags=0)
    _status()
    assert torch.equal(k2[pool.table[0, 0].item(), :, 4], kv[0, 2, :H]) and torch.equal(k2[pool.table[2, 1].item(), :, 5], kv[0, 4, :H])
    assert int((~torch.isnan(k2)).sum()) == int((~torch.isnan(pool.k)).sum()) + 3 * H * D


def test_append_reports_positions_and_pages_that_do_not_exist():
    from daisy_b200 import _lib, ops
    H = 2
    kv = _randn(_gen(1), 3, 1, 2 * H, D).cuda()
    cos, sin = (t.cuda() for t in _tables(64))

    def call(starts, table, cos_rows=64):
        k_pages = torch.full((4, H, 16, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        v_pages = k_pages.clone()
        q = ops.paged_append(kv[:, :, :H], kv[:, :, H:], k_pages, v_pages, _ints(table), _ints(starts), cos[:cos_rows], sin[:cos_rows], q=kv[:, :, :H], eps=EPS)
        return q, int((~torch.isnan(k_pages)).all(-1).sum()), int((~torch.isnan(v_pages)).all(-1).sum())
    good = [[0, 1], [2, -1], [3, -1]]
    assert call([3, 4, 5], good)[1:] == (3 * H, 3 * H)
    _status()
    assert call([3, 32, 5], good)[1:] == (2 * H, 2 * H)                # behind the table
    _status(_lib.EINVAL)
    assert call([3, 2 ** 31 - 1, 5], good)[1:] == (2 * H, 2 * H)
    _status(_lib.EINVAL)
    assert call([3, 20, 5], good)[1:] == (2 * H, 2 * H)                # an entry without a page
    _status(_lib.EINVAL)
    assert call([3, 4, 5], [[0, 1], [4, -1], [3, -1]])[1:] == (2 * H, 2 * H)
    _status(_lib.EINVAL)
    assert call([3, 20, 5], [[0, 1], [2, 2 ** 31 - 1], [3, -1]])[1:] == (2 * H, 2 * H)
    _status(_lib.EINVAL)
    assert call([3, 20, 5], [[0, 1], [2, 1], [3, -1]], cos_rows=16)[1:] == (2 * H, 2 * H)     # behind the RoPE table
    _status(_lib.EINVAL)


def test_append_value_embedding():
    from daisy_b200 import ops
    H, T = 3, 37
    pool = Pool([10, 0], [T, T], H, 32, torch.bfloat16, seed=5)
    x = _randn(_gen(6), 2, T, 3 * H, D)
    gate = torch.tensor([-0.7])
    k_pages, v_pages, table = pool.gpu()
    cos, sin = _tables()
    ops.paged_append(x[:, :, :H].cuda(), x[:, :, H:2 * H].cuda(), k_pages, v_pages, table, _ints([10, 0]), cos.cuda(), sin.cuda(), eps=EPS, ve=x[:, :, 2 * H:].cuda(),
                     ve_gate_logit=gate.cuda())
    _status()
    s = torch.sigmoid(gate.double())
    vn, ve = _norm(x[:, :, H:2 * H]), x[:, :, 2 * H:].double()
    ref = s * vn + (1 - s) * ve
    got = torch.stack([torch.stack([pool.row(v_pages.cpu(), b, p0 + i) for i in range(T)]) for b, p0 in enumerate((10, 0))])
    # the gate: e^x to 2 steps and its argument's rounding, a division and the mix, all of 2^-24: below 140 of them on |v| + |ve|
    _check(got, ref, _store_tol(ref, vn.abs() + ve.abs(), torch.bfloat16), "gated v")


# ---------------------------------------------------------------------------------------------- attention in 64 bits
def _attention(q, k, v, seen):
    """``q [n, Hq, D]``, ``k, v [H, rows, D]`` (64 bits), ``seen [n, rows]`` -> (y [n, Hq, D], sum p |v| / sum p, sum |q k| at most)."""
    G = q.shape[1] // k.shape[0]
    kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    z = torch.einsum("nhd,hrd->nhr", q, kk) * SCALE
    z = z.masked_fill(~seen[:, None], -math.inf)
    p = torch.softmax(z, -1)
    mass = torch.einsum("nhd,hrd->nhr", q.abs(), kk.abs()).masked_fill(~seen[:, None], 0).amax(-1)
    return torch.einsum("nhr,hrd->nhd", p, vv), torch.einsum("nhr,hrd->nhd", p, vv.abs()), mass


def _decode_tol(y, A, mass, rows):
    d = (2.0 ** -16 + 130 * 2.0 ** -23) * SCALE * mass[..., None]
    return 2.0 ** -8 * y.abs() + (torch.expm1(2 * d) + 2.0 ** -16 + (rows + 130) * 2.0 ** -23) * A * (1 + 2.0 ** -8)


def _attend_tol(y, A, mass, rows, dtype, vmax, bounded):
    d = 130 * 2.0 ** -23 * SCALE * mass[..., None]
    tol = 2.0 ** -8 * y.abs() + (torch.expm1(2 * d) + HALF[dtype] + (2 * 7.5e-5 if bounded else 0.0) + 2.0 ** -20 + (rows + 130) * 2.0 ** -23) * A * (1 + 2.0 ** -8)
    return tol + (rows * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0)


def _decode_case(lens, Hq, H, page, window, dtype, seed, strided=False, ve=False, workspace=None):
    from daisy_b200 import ops
    n = len(lens)
    pool = Pool(lens, [1] * n, H, page, dtype, seed, window=window, strided=strided)
    qkv = _randn(_gen(seed + 1), n, 1, Hq + 3 * H, D)
    cos, sin = _tables(max(lens) + 8)
    k_pages, v_pages, table = pool.gpu()
    before = k_pages.clone(), v_pages.clone()
    x = qkv.cuda()
    out = None
    if strided:
        out = torch.full((n, 1, Hq + 1, D + 4), 5.0, dtype=torch.bfloat16, device="cuda")[:, :, :Hq, :D]
    more = dict(ve=x[:, :, Hq + 2 * H:], ve_gate_logit=torch.tensor([0.3], device="cuda")) if ve else {}
    y = ops.paged_decode_step(x[:, :, :Hq], x[:, :, Hq:Hq + H], x[:, :, Hq + H:Hq + 2 * H], k_pages, v_pages, table, _ints(lens), window, cos.cuda(), sin.cuda(), eps=EPS, out=out,
                              workspace=workspace, **more)
    _status()
    assert out is None or y.data_ptr() == out.data_ptr()
    kc, vc = k_pages.cpu(), v_pages.cpu()
    for b, p in enumerate(lens):
        if p < 0:
            assert (y[b] == 0).all()
            continue
        pos = torch.tensor([p])
        qn, kn, vn = (_norm(t) for t in qkv[b].split([Hq, H, H, H], 1)[:3])
        if ve:
            s = torch.sigmoid(torch.tensor(0.3, dtype=torch.float64))
            mixed_v = vn.abs() + qkv[b, :, Hq + 2 * H:].double().abs()
            vn = s * vn + (1 - s) * qkv[b, :, Hq + 2 * H:].double()
        else:
            mixed_v = vn.abs()
        kr = _rotate(kn, pos, cos, sin)
        own_k, own_v = pool.row(kc, b, p), pool.row(vc, b, p)
        _check(own_k[None], kr, _store_tol(kr, _mixed(kn), dtype), f"k of {b}")
        _check(own_v[None], vn, _store_tol(vn, mixed_v, dtype), f"v of {b}")
        lo = max(0, p - window + 1) if window else 0
        k, v = pool.rows(kc, b, lo, p + 1), pool.rows(vc, b, lo, p + 1)            # with the row as it was stored
        ref, A, mass = _attention(_rotate(qn, pos, cos, sin), k, v, torch.ones(1, p + 1 - lo, dtype=torch.bool))
        # the query's own norm and rotation in 32 bits: 140 * 2^-24 on |a| + |b|, at most 2.1 |q| on the whole: inside 2^-16
        _check(y[b], ref, _decode_tol(ref, A, mass, p + 1 - lo), f"y of {b}, length {p}")
        pg, r = pool.table[b, p // page].item(), p % page
        before[0][pg, :, r], before[1][pg, :, r] = k_pages[pg, :, r], v_pages[pg, :, r]
    assert _same_bits(before[0], k_pages) and _same_bits(before[1], v_pages)
    return y


EDGES = [0, 1, 15, 16, 17, 63, 64, 65, -1, 200, 127, 128]


@pytest.mark.parametrize("window", [None, 1, 2, 16, 17, 33, 64, 5000])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_lengths_and_windows(window, page, dtype):
    _decode_case(EDGES, 2, 2, page, window, dtype, seed=11)


@pytest.mark.parametrize("Hq,H", [(1, 1), (3, 1), (4, 2), (8, 1), (9, 1), (16, 1), (20, 1), (34, 2), (24, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_head_groups(Hq, H, dtype):
    _decode_case([100, 0, 37, 530], Hq, H, 32, None, dtype, seed=21)


@pytest.mark.parametrize("strided,ve", [(True, False), (False, True), (True, True)])
def test_decode_strides_and_value_embedding(strided, ve):
    _decode_case([100, 3, -1, 64, 290], 4, 2, 32, 97, torch.bfloat16, seed=31, strided=strided, ve=ve)


def test_decode_many_sequences():
    """More sequences than a block keeps the lengths of, short and long, idle ones between."""
    lens = [(37 * b) % 23 - 1 for b in range(300)]
    lens[150], lens[299], lens[0] = 700, 90, 350
    _decode_case(lens, 1, 1, 16, None, torch.bfloat16, seed=41)


@pytest.mark.parametrize("lens,Hq,H,window", [([20000], 1, 1, None), ([20000], 12, 1, None), ([9000, 3, 30000], 2, 2, 8192)])
def test_decode_long_context_over_many_ctas(lens, Hq, H, window):
    """A pair whose shares are joined in groups."""
    _decode_case(lens, Hq, H, 256, window, torch.bfloat16, seed=51)


def test_decode_large_scores():
    """Scores far apart and far from zero: the reference maximum has to follow."""
    from daisy_b200 import ops
    H, n, page = 2, 700, 64
    pool = Pool([n], [1], H, page, torch.bfloat16, seed=61)
    grow = torch.linspace(-6, 6, n)
    for p in range(n):
        pool.row(pool.k, 0, p)[:] = (pool.row(pool.k, 0, p).float() * grow[p] * 2).bfloat16()
    x = (_randn(_gen(62), 1, 1, 3 * H, D) * 4).bfloat16()
    k_pages, v_pages, table = pool.gpu()
    y = ops.paged_decode_step(*(t.cuda() for t in x.split(H, 2)), k_pages, v_pages, table, _ints([n]), None, None, None, flags=0)
    _status()
    kc, vc = k_pages.cpu(), v_pages.cpu()
    ref, A, mass = _attention(x[0, :, :H].double(), pool.rows(kc, 0, 0, n + 1), pool.rows(vc, 0, 0, n + 1), torch.ones(1, n + 1, dtype=torch.bool))
    _check(y[0], ref, _decode_tol(ref, A, mass, n + 1), "y")


def test_decode_is_repeatable_and_workspaces_serve_all_sizes():
    from daisy_b200 import ops
    ws = ops.paged_decode_workspace(300, 64, 16, "cuda")
    first = _decode_case([20000, 77], 16, 1, 64, None, torch.bfloat16, seed=71, workspace=ws)
    for seed in range(3):                                            # other sizes through the same workspace, and through the stream's
        _decode_case([5, 90, 33], 2, 2, 16, 40, torch.bfloat16, seed=72 + seed, workspace=ws)
        _decode_case([700, 3], 8, 1, 32, None, torch.float16, seed=75 + seed)
        assert torch.equal(first, _decode_case([20000, 77], 16, 1, 64, None, torch.bfloat16, seed=71, workspace=ws))
        assert torch.equal(first, _decode_case([20000, 77], 16, 1, 64, None, torch.bfloat16, seed=71))


def test_decode_reports_what_it_cannot_reach():
    from daisy_b200 import _lib, ops
    H, page = 2, 16
    pool = Pool([40, 20, 33], [1] * 3, H, page, torch.bfloat16, seed=81, extra_entries=0)
    x = [t.cuda() for t in _randn(_gen(82), 3, 1, 3 * H, D).split(H, 2)]
    cos, sin = (t.cuda() for t in _tables(64))

    def call(lens, table, rows=64):
        k_pages, v_pages, _ = pool.gpu()
        y = ops.paged_decode_step(*x, k_pages, v_pages, table, _ints(lens), None, cos[:rows], sin[:rows], eps=EPS)
        return y, k_pages
    good, _ = call([40, 20, 33], pool.table.cuda())
    _status()
    for lens, rows in (([40, 48, 33], 64), ([40, 2 ** 31 - 1, 33], 64), ([32, 40, 33], 40)):         # behind the table, behind the RoPE table
        y, _ = call(lens, pool.table.cuda(), rows)
        _status(_lib.EINVAL)
        assert (y[1] == 0).all() and torch.isfinite(y.float()).all()
        if lens[0] == 40:
            assert torch.equal(y[0], good[0]) and torch.equal(y[2], good[2])
    for entry, bad in ((0, 10 ** 6), (1, -1), (1, -2 ** 31)):                                        # a page that the pool does not have: read, then written
        table = pool.table.clone()
        table[1, entry] = bad
        y, k_pages = call([40, 20, 33], table.cuda())
        _status(_lib.EINVAL)
        assert torch.equal(y[0], good[0]) and torch.equal(y[2], good[2])
        if entry == 1:
            assert torch.isnan(k_pages[pool.table[1, 1].item(), :, 20 % page]).all()                 # not stored


# ---------------------------------------------------------------------------------------------- chunks
def _attend_case(prior, counts, Hq, H, page, window, dtype, seed, bounded=True, packed=None, strided=False, tail=0, want_bits=None):
    from daisy_b200 import ops
    n, N = len(counts), sum(counts)
    packed = len(set(counts)) > 1 or tail > 0 if packed is None else packed
    lens = [p + c for p, c in zip(prior, counts)]
    # the cache holds the chunk already; the window of the FIRST query says what may be gone
    pool = Pool(lens, [0] * n, H, page, dtype, seed, unit=bounded)
    if window is not None:
        for b, p in enumerate(prior):
            for i in range(max(0, p - window + 1)):
                pool.row(pool.k, b, i)[:], pool.row(pool.v, b, i)[:] = float("nan"), float("inf")
            for e in range(max(0, p - window + 1) // page):
                pool.table[b, e] = -1
    g = _gen(seed + 1)
    q = torch.randn(N + tail, Hq, D, generator=g) * (1.0 if bounded else 1.5)
    if bounded:
        q = q / q.square().mean(-1, keepdim=True).sqrt()
    q = q.to(dtype)
    k_pages, v_pages, table = pool.gpu()
    before = k_pages.clone(), v_pages.clone()
    shape = (1, N + tail) if packed else (n, counts[0])
    x = q.cuda().unflatten(0, shape)
    out = None
    if strided or tail:
        x = torch.cat([x, x.roll(1, -1)], 2)[:, :, :Hq]
        out = torch.full((*shape, Hq + 1, D), 9.0, dtype=torch.bfloat16, device="cuda")[:, :, :Hq]
    cu = _ints([sum(counts[:i]) for i in range(n + 1)]) if packed else None
    y = ops.paged_attend(x, k_pages, v_pages, table, _ints(lens), window, cu_seqlens=cu, bounded_qk=bounded, out=out)
    _status()
    assert y.shape == x.shape and y.dtype == torch.bfloat16 and _same_bits(before[0], k_pages) and _same_bits(before[1], v_pages)
    y = y.flatten(0, 1)
    if tail:
        assert (y[N:] == 9.0).all()                                  # tokens of nobody
    few = max(counts) * (Hq // H) <= 8 and N * (Hq // H) <= 32
    at = 0
    for b, (p, c) in enumerate(zip(prior, counts)):
        lo = max(0, p - window + 1) if window else 0
        k, v = pool.rows(pool.k, b, lo, p + c), pool.rows(pool.v, b, lo, p + c)
        gap = (p + torch.arange(c))[:, None] - torch.arange(lo, p + c)[None]
        seen = (gap >= 0) & ((gap < window) if window else torch.ones_like(gap, dtype=torch.bool))
        if c:
            ref, A, mass = _attention(q[at:at + c].double(), k, v, seen)
            # (a few queries go by the decode step's arithmetic, whose tolerance is the smaller one)
            _check(y[at:at + c], ref, _attend_tol(ref, A, mass, p + c - lo, dtype, v.abs().max(), bounded and dtype == torch.bfloat16), f"sequence {b}, few={few}")
        at += c
    return y


@pytest.mark.parametrize("prior,counts", [([0], [1]), ([0], [127]), ([0], [129]), ([5], [300]), ([128], [128]), ([1, 500], [257, 257]), ([0, 130, 7, 64], [3, 200, 0, 90]),
                                          ([9] * 31 + [300], [11] * 31 + [140]), ([9] * 33, [5] * 32 + [30]), ([700], [40]), ([255, 256, 257], [9, 9, 9])])
@pytest.mark.parametrize("window", [None, 1, 50, 128, 300])
@pytest.mark.parametrize("dtype,bounded", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, True)])
def test_attend(prior, counts, window, dtype, bounded):
    _attend_case(prior, counts, 2, 2, 64, window, dtype, seed=91, bounded=bounded)


@pytest.mark.parametrize("page", [16, 32, 128, 256])
@pytest.mark.parametrize("dtype,bounded", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
def test_attend_pages(page, dtype, bounded):
    _attend_case([0, 130, 61], [300, 20, 150], 2, 1, page, 170, dtype, seed=101, bounded=bounded)


@pytest.mark.parametrize("Hq,H", [(1, 1), (2, 1), (3, 1), (4, 1), (6, 1), (8, 2), (12, 1), (16, 1), (32, 1), (10, 2)])
@pytest.mark.parametrize("bounded", [True, False])
def test_attend_head_groups(Hq, H, bounded):
    _attend_case([40, 200], [33, 50], Hq, H, 32, 190, torch.bfloat16, seed=111, bounded=bounded)


@pytest.mark.parametrize("prior,counts,Hq,H", [([0], [1], 1, 1), ([300, 20, 0, 64], [4, 4, 4, 4], 2, 1), ([17, 900, 3, 100, 0, 63, 64, 65], [1, 5, 2, 0, 3, 4, 4, 3], 2, 2),
                                               ([100, 5, 33, 8], [2, 2, 2, 2], 8, 2), ([250, 4, 31, 9, 77, 60, 3, 2], [20, 1, 1, 1, 2, 1, 1, 1], 1, 1), ([5000], [8], 1, 1)])
@pytest.mark.parametrize("window", [None, 1, 3, 60])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_few_queries(prior, counts, Hq, H, window, dtype):
    from daisy_b200 import _lib
    packed = len(set(counts)) > 1
    if (Hq, H) != (8, 2):
        assert _lib.lib().daisy_b200_paged_attend_few_rows(sum(counts) if packed else counts[0], len(counts), int(packed), Hq, H) > 0
    _attend_case(prior, counts, Hq, H, 16, window, dtype, seed=121, bounded=False)


@pytest.mark.parametrize("prior,counts,Hq,H,window", [([9000], [20], 2, 2, None), ([6000, 50], [130, 300], 4, 1, None), ([20000], [9], 1, 1, None), ([5000, 9000, 100], [60, 10, 400], 1, 1, 4000)])
@pytest.mark.parametrize("dtype,bounded", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
def test_attend_long_contexts_are_cut(prior, counts, Hq, H, window, dtype, bounded):
    """Few items with long contexts go in pieces: joined in a fixed order, the same bits every time."""
    a = _attend_case(prior, counts, Hq, H, 64, window, dtype, seed=131, bounded=bounded)
    assert torch.equal(a, _attend_case(prior, counts, Hq, H, 64, window, dtype, seed=131, bounded=bounded))


@pytest.mark.parametrize("counts", [[7 * b % 12 for b in range(1300)], [9] * 1100])
@pytest.mark.parametrize("longest", [200, 2500])
@pytest.mark.parametrize("bounded", [True, False])
def test_attend_many_sequences(counts, longest, bounded):
    """More sequences than a warp counts, more items than the plan keeps; with and without a table long enough for a plan."""
    prior = [31 * b % 40 for b in range(len(counts))]
    prior[700] = longest
    _attend_case(prior, counts, 1, 1, 16, None, torch.bfloat16, seed=136, bounded=bounded)


@pytest.mark.parametrize("T", [2400, 2560, 2720])
@pytest.mark.parametrize("dtype,bounded", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
def test_attend_items_left_over_by_whole_rounds(T, dtype, bounded):
    """150 to 170 items of like length: a few more than there are SMs, so that the last ones are cut."""
    from daisy_b200 import ops
    Hq, page, prior, window = 16, 64, 2300, 2000
    pool = Pool([prior + T], [0], 1, page, dtype, seed=137)
    q = torch.randn(1, T, Hq, D, generator=_gen(138))
    q = (q / q.square().mean(-1, keepdim=True).sqrt()).to(dtype)
    k_pages, v_pages, table = pool.gpu()
    y = ops.paged_attend(q.cuda(), k_pages, v_pages, table, _ints([prior + T]), window, bounded_qk=bounded)
    assert torch.equal(y, ops.paged_attend(q.cuda(), k_pages, v_pages, table, _ints([prior + T]), window, bounded_qk=bounded))
    _status()
    k, v = pool.rows(pool.k, 0, 0, prior + T), pool.rows(pool.v, 0, 0, prior + T)
    for at in [*range(0, T, 300), T - 200, T - 90, T - 10]:          # ten queries here and there
        own = prior + torch.arange(at, at + 10)
        gap = own[:, None] - torch.arange(prior + T)[None]
        ref, A, mass = _attention(q[0, at:at + 10].double(), k, v, (gap >= 0) & (gap < window))
        _check(y[0, at:at + 10], ref, _attend_tol(ref, A, mass, window, dtype, v.abs().max(), bounded), f"queries from {at}")


@pytest.mark.parametrize("few", [False, True])
def test_attend_strides_and_tokens_of_nobody(few):
    counts = [1, 2, 3] if few else [30, 0, 150]
    _attend_case([10, 70, 128], counts, 2, 2, 32, 100, torch.bfloat16, seed=141, strided=True, tail=5)
    _attend_case([10, 70, 128], [4 if few else 140] * 3, 2, 2, 32, None, torch.bfloat16, seed=142, strided=True)


@pytest.mark.parametrize("T", [3, 40])
def test_attend_idle_and_refused_sequences(T):
    from daisy_b200 import _lib, ops
    H, page = 2, 16
    pool = Pool([60, 60, 60, 60], [0] * 4, H, page, torch.bfloat16, seed=151, extra_entries=0)
    q = _norm(torch.randn(4, T, H, D, generator=_gen(152))).bfloat16().cuda()
    k_pages, v_pages, table = pool.gpu()

    def call(lens, table=table):
        return ops.paged_attend(q, k_pages, v_pages, table, _ints(lens), None, bounded_qk=True)
    good = call([60, 60, 60, 60])
    _status()
    y = call([60, -1, 60, 60])                                       # idle: no complaint
    _status()
    assert (y[1] == 0).all() and torch.equal(y[[0, 2, 3]], good[[0, 2, 3]])
    for bad in (T - 1, 65, 2 ** 31 - 1, 0):                          # fewer tokens than queries, more than the table holds
        y = call([60, 60, bad, 60])
        _status(_lib.EINVAL)
        assert (y[2] == 0).all() and torch.equal(y[[0, 1, 3]], good[[0, 1, 3]])
    for bad in (-1, 10 ** 6):                                        # a page that the pool does not have is read as page 0
        t2 = pool.table.clone()
        t2[3, 1] = bad
        t3 = pool.table.clone()
        t3[3, 1] = 0
        y = call([60, 60, 60, 60], t2.cuda())
        _status(_lib.EINVAL)
        assert torch.equal(y[:3], good[:3])
    # offsets that decrease or leave the row: those sequences have no queries
    out = torch.full((1, 4 * T, H, D), 3.0, dtype=torch.bfloat16, device="cuda")
    y = ops.paged_attend(q.flatten(0, 1)[None], k_pages, v_pages, table, _ints([60] * 4), None, cu_seqlens=_ints([0, T, 0, 2 * T, 9 * T]), bounded_qk=True, out=out)
    _status(_lib.EINVAL)
    assert torch.isfinite(y.float()).all() and (y[0, 2 * T:] == 3.0).all()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 40, 200])
@pytest.mark.parametrize("T", [3, 150])
@pytest.mark.parametrize("bounded", [True, False])
def test_windows_longer_than_any_sequence_are_none(window, T, bounded):
    from daisy_b200 import ops
    H, page, lens = 2, 16, [160, 190]
    pool = Pool(lens, [1, 1], H, page, torch.bfloat16, seed=155, extra_entries=0)
    q = _norm(torch.randn(2, T, H, D, generator=_gen(156))).bfloat16().cuda()
    x = [t.cuda() for t in _randn(_gen(157), 2, 1, 3 * H, D).split(H, 2)]
    cos, sin = (t.cuda() for t in _tables(200))
    got = []
    for w in (window, None):
        k_pages, v_pages, table = pool.gpu()
        got.append((ops.paged_attend(q, k_pages, v_pages, table, _ints(lens), w, bounded_qk=bounded),
                    ops.paged_decode_step(*x, k_pages, v_pages, table, _ints(lens), w, cos, sin, eps=EPS)))
    _status()
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_offsets_past_32_bits():
    """Pages whose element offsets need more than 32 bits."""
    from daisy_b200 import ops
    H, page = 2, 256
    per_page = H * page * D
    pages = 2 ** 32 // per_page + 3                                  # 8.6 GB a pool
    k_pages = torch.empty(pages, H, page, D, dtype=torch.bfloat16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    lens, n = [300, 20], 40
    pool = Pool(lens, [n + 1] * 2, H, page, torch.bfloat16, seed=161, spare=0, extra_entries=0)
    far = [pages - 1, pages - 2, pages - 3, 2 ** 31 // per_page]
    table = pool.table.clone()
    for i in range(pool.k.shape[0]):
        table[pool.table == i] = far[i]
        k_pages[far[i]], v_pages[far[i]] = pool.k[i].cuda(), pool.v[i].cuda()
    near = pool.gpu()
    x = _randn(_gen(162), 2, n, 3 * H, D).cuda()
    y1 = _randn(_gen(163), 2, 1, 3 * H, D).cuda()
    cos, sin = (t.cuda() for t in _tables())
    got = []
    for k, v, t in ((k_pages, v_pages, table.cuda()), near):
        q = ops.paged_append(x[:, :, H:2 * H], x[:, :, 2 * H:], k, v, t, _ints(lens), cos, sin, q=x[:, :, :H], eps=EPS)
        a = ops.paged_attend(q, k, v, t, _ints([m + n for m in lens]), None, bounded_qk=True)
        f = ops.paged_attend(q[:, -3:], k, v, t, _ints([m + n for m in lens]), None, bounded_qk=True)
        d = ops.paged_decode_step(*y1.split(H, 2), k, v, t, _ints([m + n for m in lens]), None, cos, sin, eps=EPS)
        got.append((q, a, f, d))
    _status()
    for far_x, near_x in zip(*got):
        assert torch.equal(far_x, near_x)
    for i in range(pool.k.shape[0]):
        assert _same_bits(k_pages[far[i]], near[0][i]) and _same_bits(v_pages[far[i]], near[1][i])


# ---------------------------------------------------------------------------------------------- together
def test_append_then_attend_on_another_stream_and_captured():
    """The calls of a step recorded once and replayed on another stream while the lengths move, against eager calls."""
    from daisy_b200 import ops
    H, page, lens = 4, 16, [30, 0, 100]
    pool = Pool(lens, [40] * 3, H, page, torch.bfloat16, seed=171)
    cos, sin = (t.cuda() for t in _tables())
    tokens = [_randn(_gen(172 + i), 3, 3, 3 * H, D).cuda() for i in range(6)]
    eager = pool.gpu()
    want, pos = [], list(lens)
    for x in tokens:
        q = ops.paged_append(x[:, :, H:2 * H], x[:, :, 2 * H:], *eager, _ints(pos), cos, sin, q=x[:, :, :H], eps=EPS)
        a = ops.paged_attend(q, *eager, _ints([p + 3 for p in pos]), 60, bounded_qk=True)
        d = ops.paged_decode_step(*x[:, :1].split(H, 2), *eager, _ints([p + 3 for p in pos]), 60, cos, sin, eps=EPS)
        pos = [p + 4 for p in pos]
        want.append((q, a, d))
    mine = pool.gpu()
    x, start = torch.zeros_like(tokens[0]), _ints(lens)

    def body():
        q = ops.paged_append(x[:, :, H:2 * H], x[:, :, 2 * H:], *mine, start, cos, sin, q=x[:, :, :H], eps=EPS)
        after = start + 3
        a = ops.paged_attend(q, *mine, after, 60, bounded_qk=True)
        d = ops.paged_decode_step(*x[:, :1].split(H, 2), *mine, after, 60, cos, sin, eps=EPS)
        start.add_(4)
        return q, a, d
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        start.fill_(-10)
        body()                                                       # idle, also three tokens on: warms up, stores nothing
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = body()
    start.copy_(_ints(lens))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for x_new, w in zip(tokens, want):
        with torch.cuda.stream(other):
            x.copy_(x_new)
            graph.replay()
        eager_again = ops.paged_attend(w[0], *eager, _ints([p + 3 for p in lens]), 60, bounded_qk=True)      # beside it, on the current stream
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))
        del eager_again
    _status()
    assert _same_bits(mine[0], eager[0]) and _same_bits(mine[1], eager[1])


def _stack(L, H, dim):
    from daisy_b200 import B200CausalSelfAttention
    torch.manual_seed(5)
    layers = []
    for _ in range(L):
        a = B200CausalSelfAttention(dim, H, D, max_seq_len=2048)
        with torch.no_grad():
            a.qkvo_w.copy_(torch.randn(4, dim, dim) * dim ** -0.5)
        layers.append(a.cuda())
    return layers


def test_runner_refusals():
    from daisy_b200 import PagedRunner
    dim = 2 * D
    runner = PagedRunner(_stack(1, 2, dim), 50, pages=4, max_seqs=2, max_len=100, page=32)
    x = torch.zeros(2, 1, dim, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):                                # nothing recorded
        runner.step_graph(x)
    runner.capture_step(dim)
    slot = runner.add()
    for bad in (x[:1], x[0]):
        with pytest.raises(ValueError):
            runner.step_graph(bad)
    with pytest.raises(RuntimeError):                                # a sequence is there
        runner.capture_step(dim)
    with pytest.raises(ValueError):
        runner.prefill([x[0], x[1]], [slot, slot])
    with pytest.raises(ValueError):                                  # more than the table holds
        runner.prefill([torch.zeros(101, dim, dtype=torch.bfloat16, device="cuda")], [slot])
    assert runner.cache.length == [0, -1] and len(runner.cache.book.free) == 4
    _status()


@pytest.mark.parametrize("window,page", [(None, 16), (90, 32), (33, 64)])
@pytest.mark.parametrize("graph", [False, True])
def test_runner_serves_sequences_that_come_and_go(window, page, graph):
    """Prompts in pieces and steps of three sequences, one of which ends while another begins, against the dense layers over each whole
    sequence; pages behind the window are given back."""
    from daisy_b200 import PagedRunner, WindowMask
    H, L = 2, 2
    dim = H * D
    layers = _stack(L, H, dim)
    runner = PagedRunner(layers, window, pages=60, max_seqs=3, max_len=700, page=page)
    if graph:
        runner.capture_step(dim)
    g = _gen(181)
    fed, got = {}, {}

    def prompt(names, counts):
        xs = [torch.randn(n, dim, generator=g).bfloat16().cuda() for n in counts]
        for name in names:
            if name not in fed:
                fed[name], got[name] = [], []
                slot[name] = runner.add()
        ys = runner.prefill(xs, [slot[name] for name in names])
        for name, x, y in zip(names, xs, ys):
            fed[name].append(x)
            got[name].append(y.clone())

    def steps(names, n):
        for _ in range(n):
            x = torch.randn(3, 1, dim, generator=g).bfloat16().cuda()
            y = (runner.step_graph if graph else runner.step)(x)
            for name in names:
                fed[name].append(x[slot[name]])
                got[name].append(y[slot[name]].clone())
    slot = {}
    prompt(["a", "b"], [150, 3])
    steps(["a", "b"], 5)
    assert [y.shape for y in runner.prefill([torch.zeros(0, dim, dtype=torch.bfloat16, device="cuda")] * 2, [0, 1])] == [(0, dim)] * 2
    prompt(["b"], [70])
    prompt(["c", "a"], [300, 4])
    steps(["a", "b", "c"], 40)
    runner.drop(slot["b"])
    steps(["a", "c"], 3)
    prompt(["d"], [129])
    steps(["a", "c", "d"], 6)
    _status()
    c = runner.cache
    assert c.lens.tolist() == c.length
    for name in "abcd":
        x = torch.cat(fed[name])[None]
        for a in layers:
            with torch.inference_mode():
                x, _, _ = a.prefill(x, None, attn_mask=WindowMask(window))
        assert_close_bf16(torch.cat(got[name]), x[0], f"sequence {name}")
    if window:
        held = sum(p >= 0 for row in c.book.table for p in row)
        assert held <= 3 * (-(-window // page) + 1) and held + len(c.book.free) == 60
    for name in "acd":
        runner.drop(slot[name])
    assert sorted(c.book.free) == list(range(60)) and c.lens.tolist() == [-1] * 3
    with pytest.raises(RuntimeError, match="pages left"):
        s = runner.add()
        runner.prefill([torch.zeros(700, dim, dtype=torch.bfloat16, device="cuda")] * 2, [s, runner.add()]) if page == 16 else runner.cache.book.reserve([s], [700]) and \
            [runner.cache.book.free.clear(), runner.cache.reserve([runner.add()], 1)]


def test_layer_with_a_value_embedding():
    """A gated layer's paged calls against its dense ones."""
    from daisy_b200 import B200CausalSelfAttention, B200PagedKVCache, WindowMask
    H, dim, T, window = 2, 256, 140, 50
    torch.manual_seed(9)
    a = B200CausalSelfAttention(dim, H, D, receives_ve=True, layer_idx=0, max_seq_len=512)
    with torch.no_grad():
        a.qkvo_w.copy_(torch.randn(4, dim, dim) * dim ** -0.5)
    a = a.cuda()
    x, ve = (torch.randn(1, T + 1, dim, generator=_gen(s)).bfloat16().cuda() for s in (191, 192))
    with torch.inference_mode():
        ref, _, _ = a.prefill(x, ve, attn_mask=WindowMask(window))
        cache = B200PagedKVCache(1, 12, H, D, 1, 256, "cuda", page=16)
        slot = cache.claim()
        cache.reserve([slot], T + 1)
        y = a.prefill_paged(x[:, :T], ve[:, :T], cache, 0, cache.table, _ints([0]), _ints([T]), window)
        cache.advance([slot], T)
        y1 = a.step_paged(x[:, T:], ve[:, T:], cache, 0, window)
    _status()
    assert_close_bf16(torch.cat([y, y1], 1), ref, "gated layer")


def test_refusals():
    from daisy_b200 import ops
    pool, x, ids = torch.zeros(4, 2, 16, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, 2, D, dtype=torch.bfloat16, device="cuda"), _ints([[0, 1]])
    cos, sin = (t.cuda() for t in _tables(32))
    one = _ints([3])
    step = lambda q=x, k=x, kp=pool, vp=pool, t=ids, n=one, **kw: ops.paged_decode_step(q, k, x, kp, vp, t, n, None, cos, sin, **kw)
    step()
    for error, kw in ((TypeError, dict(q=x.half())), (ValueError, dict(q=x[:, :, :, :64])), (ValueError, dict(q=x.expand(1, 2, 2, D))), (ValueError, dict(k=x[:, :, :1])),
                      (TypeError, dict(kp=pool.float(), vp=pool.float())), (TypeError, dict(vp=pool.half())), (ValueError, dict(kp=pool[:, :, :12], vp=pool[:, :, :12])),
                      (ValueError, dict(t=ids[0])), (TypeError, dict(t=ids.long())), (TypeError, dict(n=one.long())), (ValueError, dict(n=_ints([1, 2]))), (ValueError, dict(n=one.cpu())),
                      (ValueError, dict(flags=64)), (ValueError, dict(ve=x)), (ValueError, dict(out=torch.zeros(1, 2, D, dtype=torch.bfloat16, device="cuda"))),
                      (ValueError, dict(workspace=torch.zeros(4, device="cuda"))), (RuntimeError, dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))),
                      (ValueError, dict(t=torch.stack([ids[0], ids[0]], -1)[:, 0][None]))):
        with pytest.raises(error):
            step(**kw)
    with pytest.raises(ValueError):
        ops.paged_attend(x.expand(2, 1, 2, D), pool, pool, ids, one, None)                           # one sequence, two rows
    with pytest.raises(ValueError):
        ops.paged_attend(x.expand(2, 1, 2, D), pool, pool, ids, one, None, cu_seqlens=_ints([0, 1]))
    with pytest.raises(TypeError):
        ops.paged_attend(x.half(), pool, pool, ids, one, None)                                       # queries are of the pages' type
    with pytest.raises(ValueError):
        ops.paged_attend(x[:, :, :1].expand(1, 1, 3, D), pool, pool, ids, one, None)                 # 3 heads over 2
    with pytest.raises(ValueError):
        ops.paged_append(x, x, pool, pool, ids, one, None, sin, q=x)                                 # a rotation without a table
    with pytest.raises(ValueError):
        ops.paged_append(x, x, pool, pool, ids, one, cos, sin, q=torch.zeros(1, 2, 2, D, dtype=torch.bfloat16, device="cuda"))
    empty = torch.zeros(1, 0, 2, D, dtype=torch.bfloat16, device="cuda")
    assert ops.paged_append(empty, empty, pool, pool, ids, one, cos, sin, q=empty).shape == empty.shape
    assert ops.paged_attend(empty, pool, pool, ids, one, None).shape == empty.shape
    _status()
