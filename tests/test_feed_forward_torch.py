"""Host logic of the feed-forward operators on torch tensors, without a device: CPU tensors that say they
lie on cuda:0, and launches that are written down instead of made.  Checks of arguments, and what every
launch is told of its operands."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from triton_metal import cuda, functional  # noqa: E402


class OnCuda(torch.Tensor):
    """A CPU tensor that passes for one of cuda:0 (so do the results of its methods)."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 0))


def on_cuda(t):
    return t.as_subclass(OnCuda)


@pytest.fixture()
def calls(monkeypatch):
    """The launches made: dicts of the kernel's name, values and lengths by argument name."""
    made = []

    def record(handle, stream, gx, gy, gz, threads, kinds, values, lengths, n):
        kern = next(k for k in functional._KERNELS.values() if k.handle == handle)
        unpack = lambda b: dict(zip(kern.names, memoryview(b).cast("q").tolist()))  # noqa: E731
        assert n == len(kern.names) and isinstance(kinds, ctypes.Array)
        made.append(dict(name=kern.name, values=unpack(values), lengths=unpack(lengths)))
        return 0

    monkeypatch.setattr(cuda, "get_device", lambda: 0)
    monkeypatch.setattr(functional, "_launch_on", record)
    monkeypatch.setattr(functional, "_raw_stream", lambda index: 0)
    functional.release()
    yield made
    functional.release()


def zeros(*shape, dtype=torch.bfloat16):
    return on_cuda(torch.zeros(*shape, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_row_statistics_are_float32_whatever_the_operands_are(calls, dtype):
    """Four fp32 words a row are read: statistics of a 16-bit type would be read past their end."""
    M, D = 6, 64
    dn, s, w = zeros(M, D, dtype=dtype), zeros(M, D, dtype=dtype), zeros(D, dtype=dtype)
    functional.residual_norm_backward(dn, None, s, zeros(M, 4, dtype=torch.float32), w)
    assert len(calls) == 1 and calls[0]["lengths"]["stats"] == M * 4 * 4
    assert calls[0]["lengths"]["sum"] == M * D * s.element_size()
    for other in (torch.bfloat16, torch.float16, torch.float64):
        with pytest.raises(TypeError, match="stats is torch.(bfloat16|float16|float64), expected torch.float32"):
            functional.residual_norm_backward(dn, None, s, zeros(M, 4, dtype=other), w)
    assert len(calls) == 1
