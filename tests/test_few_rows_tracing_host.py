"""CPU: a traced call that quantises or dequantises 4-bit weights records the registered op, and runs it again on new inputs.  The C
calls are replaced by ones that fill their outputs with a number of their own."""

import contextlib
import ctypes

import pytest
import torch

from primus_turbo_b200 import _lib
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.kernels import few_rows_impl
from primus_turbo_b200.pytorch.ops import dequantize_int4, int4, quantize_int4

BF = torch.bfloat16


@pytest.fixture
def fake_calls(monkeypatch):
    """Every call lands in the list; the n-th fills what it writes with bytes of n."""
    calls = []

    def call(name, *a):
        calls.append(name)
        if name == "ptb_dequant_int4":
            rows, k, out = a[3], a[4], a[6]
            ctypes.memset(out, len(calls), rows * k * 2)
        else:
            rows, k, group, codes, scale, zero = a[2], a[3], a[4], a[5], a[6], a[7]
            ctypes.memset(codes, len(calls), rows * -(-k // 128) * 64)
            ctypes.memset(scale, len(calls), rows * -(-k // group) * 2)
            if zero is not None:
                ctypes.memset(zero, len(calls), rows * -(-k // group))

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(few_rows_impl, "stream_of", lambda t: 0)
    monkeypatch.setattr(int4, "require_cuda", lambda *t: None)
    return calls


def _bytes(t):
    return t.contiguous().view(torch.uint8).unique().tolist()


def test_a_traced_dequantise_runs_again(fake_calls):
    w = Int4Weight.from_codes(torch.zeros(16, 64, dtype=torch.uint8), torch.ones(16, 1, dtype=BF), group_size=64)
    traced = torch.jit.trace(lambda x: (dequantize_int4(w), x + 1), (torch.zeros(2),), check_trace=False)
    assert "dequant_int4" in str(traced.graph)
    before = len(fake_calls)
    values, _ = traced(torch.zeros(2))
    assert len(fake_calls) == before + 1 and _bytes(values) == [before + 1]


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("shape", [(16, 200), (2, 8, 64)])
def test_a_traced_quantise_runs_again(fake_calls, symmetric, shape):
    def f(x):
        q = quantize_int4(x, 32, symmetric)
        return (q.qdata, q.scale) if symmetric else (q.qdata, q.scale, q.zero)

    traced = torch.jit.trace(f, (torch.zeros(shape, dtype=BF),), check_trace=False)
    assert "quant_int4" in str(traced.graph)
    before = len(fake_calls)
    for part in traced(torch.zeros(shape, dtype=BF)):
        assert _bytes(part) == [before + 1]
    assert len(fake_calls) == before + 1
