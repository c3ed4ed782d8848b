"""Calls of the paged cache at the borders of what its documentation allows, against the formula in 64 bits.  Tolerances as in
``test_gpu_paged``; what a case adds to them stands beside it."""
import math

import pytest
import torch

from test_gpu_paged import D, EPS, SCALE, _attend_tol, _decode_tol, _gen, _ints, _randn, _status, _tables

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
