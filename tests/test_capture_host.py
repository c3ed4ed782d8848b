"""Recordings are made on the device of what they read, whichever is the current one."""
import contextlib
import types

import pytest
import torch

from daisy_b200 import PagedRunner, StepRunner, generate, kda
from daisy_b200.kda import B200KimiLinearSelfAttention


@pytest.fixture
def recorded(monkeypatch):
    """Stands in for CUDA's streams and graphs: notes the device of the stream that each recording is made on (None: the current device's)."""
    class Stream:
        def __init__(self, device=None):
            self.device = device

        def wait_stream(self, other):
            pass
    seen = []

    @contextlib.contextmanager
    def graph(g, stream=None, **kw):
        seen.append(None if stream is None else stream.device)
        yield
    for name, value in (("Stream", Stream), ("current_stream", Stream), ("stream", lambda s: contextlib.nullcontext()), ("CUDAGraph", object), ("graph", graph)):
        monkeypatch.setattr(torch.cuda, name, value)
    return seen


DEV = torch.device("cpu")            # a device that is not the current CUDA device


def test_paged_runner(recorded, monkeypatch):
    monkeypatch.setattr(generate.ops, "paged_decode_workspace", lambda *a: None)
    r = object.__new__(PagedRunner)
    r.layers, r.window = [], None
    r.cache = types.SimpleNamespace(length=[-1], device=DEV, max_seqs=1, H=1, lens=torch.zeros(1), active=torch.zeros(1))
    r.capture_step(16)
    assert recorded == [DEV]


def test_step_runner(recorded, monkeypatch):
    r = object.__new__(StepRunner)
    r.layers, r.window = [], 4
    r.cache = types.SimpleNamespace(device=DEV, t_dev=torch.zeros(1, dtype=torch.int64))
    monkeypatch.setattr(StepRunner, "_one_launch", lambda self, x: False)
    r.capture_step(1, 16)
    assert recorded == [DEV]


def test_kimi_layer(recorded, monkeypatch):
    monkeypatch.setattr(kda, "ext", lambda: types.SimpleNamespace(kda_token_supported=lambda h: False))
    monkeypatch.setattr(B200KimiLinearSelfAttention, "_forward_core", lambda self, x, *a, **k: x)
    layer = object.__new__(B200KimiLinearSelfAttention)
    torch.nn.Module.__init__(layer)
    layer.hidden_size, layer.num_heads, layer.use_short_conv, layer._conv_state, layer._seen = 16, 1, False, None, 0
    layer._recurrent_state = torch.zeros(1, 1, 4, 4)
    layer.capture_step(1)
    assert recorded == [DEV]
