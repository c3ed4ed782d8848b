"""KDA's two passes beside one another, many times: the same bits every time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_kda_parts_repeat_bit_for_bit():
    """20,000 calls of 64 rows in three parts, L2 cold before each, so that the state's pass waits for memory while the next part's pass runs: a
    stage of its ring that is refilled too early shows in the outputs (it did once in 20,000 to 70,000 calls)."""
    from daisy_b200 import _lib, ops
    lib = _lib.lib()
    B, T, H = 4, 64 * 60 + 33, 16
    g_ = torch.Generator("cuda").manual_seed(11)
    q, k, v = (torch.randn(B, T, H, 128, generator=g_, device="cuda").bfloat16() for _ in range(3))
    g = torch.nn.functional.logsigmoid(torch.randn(B, T, H, 128, generator=g_, device="cuda"))
    beta = torch.sigmoid(torch.randn(B, T, H, generator=g_, device="cuda"))
    ws = torch.empty(lib.daisy_b200_kda_workspace_bytes(B, T, H, 128, 128), dtype=torch.uint8, device="cuda")
    out = [torch.empty_like(q) for _ in range(8)]
    cold = torch.empty(160 << 20, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def call(o):
        _lib.check(lib.daisy_b200_kda_chunk_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), None, o.data_ptr(), None, B, T, H, 128, 128, 64, 0.0, 1, ws.data_ptr(),
                                                ws.numel(), None, stream), "kda")
    call(out[0])
    want = out[0].clone()
    bad = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(2500):
        for o in out:
            cold.zero_()
            call(o)
        bad += torch.stack([(o != want).any() for o in out]).sum()
    ops.check_device_status("cuda")
    assert bad.item() == 0
