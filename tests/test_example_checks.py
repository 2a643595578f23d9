"""The comparisons that the example layers make of their own results, with stand-ins for the layer on the CPU: results that
are not numbers are as far from the formula as can be."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from examples import fp8_layer, paged_decode  # noqa: E402


class OnTheCpu:
    """torch, whose new tensors are the CPU's whatever device is asked for."""

    def __getattr__(self, name):
        value = getattr(torch, name)
        if name not in ("empty", "full", "tensor", "zeros"):
            return value
        return lambda *args, device=None, **options: value(*args, **options)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self: self)
    for example in (fp8_layer, paged_decode):
        monkeypatch.setattr(example, "torch", OnTheCpu())


def spoiled(shape, value, dtype):
    """Ones, and `value` in the last place."""
    out = torch.ones(shape, dtype=dtype)
    out.view(-1)[-1] = value
    return out


VALUES = [1.0, 1.5, math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("spoil", ["out", "stream"])
def test_fp8_layer(on_cpu, monkeypatch, spoil, value):
    class Layer:
        left = torch.tensor([0])

        def __init__(self, **options):
            pass

        def step(self, y, r, counts, lengths, table):
            out, stream = (spoiled(y.shape, value if name == spoil else 1.0, t) for name, t in
                           (("out", torch.float16), ("stream", torch.float32)))
            return out, stream, lengths, table

    monkeypatch.setattr(fp8_layer, "Layer", Layer)
    monkeypatch.setattr(fp8_layer, "formula", lambda layer, x, new: (torch.ones((new, x.shape[1]), dtype=torch.float64),) * 2)
    worst = fp8_layer.run(requests=2, steps=1, hidden=16)
    assert worst == (0.0 if value == 1.0 else 0.5 / 4 if value == 1.5 else math.inf)  # (a decode step's 16 values)


@pytest.mark.parametrize("value", VALUES)
def test_paged_decode(on_cpu, monkeypatch, value):
    class Layer:
        left = torch.tensor([0])

        def __init__(self, **options):
            pass

        def step(self, x, counts, lengths, start, table, prefix):
            return None, spoiled((len(x), 2, 4), value, torch.float16), lengths, table

    def formula(layer, x, new):
        return torch.ones((new, 2, 4), dtype=torch.float64), torch.full((new, 2, 4), 0.25, dtype=torch.float64)

    monkeypatch.setattr(paged_decode, "Layer", Layer)
    monkeypatch.setattr(paged_decode, "formula", formula)
    worst = paged_decode.run(requests=2, steps=1, prefix=3, hidden=16)
    assert worst == (0.0 if value == 1.0 else 2.0 if value == 1.5 else math.inf)


def test_fp8_layer_as_a_program(monkeypatch):
    """Results that are all zero are off by 1, a part of the layer left out by less: its exit status tells."""
    for worst, status in ((0.0, 0), (0.2, 0), (0.25, 1), (0.9, 1), (1.0, 1), (math.inf, 1), (math.nan, 1)):
        monkeypatch.setattr(fp8_layer, "run", lambda **options: worst)
        assert fp8_layer.main(["--requests", "1"]) == status
