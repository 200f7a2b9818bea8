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


def operator_calls(x, w, g):
    """Every function once, on 64 x 64 operands (w also as a vector's source)."""
    stats = on_cuda(torch.zeros(64, 4))
    return {
        "linear": lambda: functional.linear(x, w, activation="silu"),
        "linear_backward": lambda: functional.linear_backward(g, x, w),
        "gated_linear": lambda: functional.gated_linear(x, w, w),
        "gated_linear_backward": lambda: functional.gated_linear_backward(g, x, w, w, g, g),
        "residual_norm": lambda: functional.residual_norm(x, g, w[0]),
        "residual_norm_backward": lambda: functional.residual_norm_backward(g, None, x, stats, w[0]),
    }


@pytest.mark.parametrize("name", sorted(operator_calls(None, None, None)))
@pytest.mark.parametrize("which", ["x", "w"])
def test_an_operand_that_requires_grad_is_refused(calls, name, which):
    """The functions record no graph: with grad mode on, the operand's gradient would be missing without a word."""
    t = {k: zeros(64, 64, dtype=torch.float32) for k in "xwg"}
    call = lambda: operator_calls(**t)[name]()  # noqa: E731
    call()
    made = len(calls)
    t[which] = t[which].clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="requires grad, and these functions record no graph"):
        call()
    assert len(calls) == made
    with torch.no_grad():
        call()
    with torch.inference_mode():
        call()
    assert len(calls) == 3 * made
    t[which] = t[which].detach()
    call()


def test_a_forward_mode_tangent_is_refused(calls):
    from torch.autograd import forward_ad
    x, w = zeros(8, 16, dtype=torch.float32), zeros(16, 24, dtype=torch.float32)
    functional.linear(x, w)
    with forward_ad.dual_level():
        functional.linear(x, w)
        dual = forward_ad.make_dual(x, torch.ones(8, 16).as_subclass(OnCuda))
        for grad_mode in (torch.no_grad, torch.enable_grad):
            with grad_mode(), pytest.raises(RuntimeError, match="x carries a forward-mode tangent"):
                functional.linear(dual, w)
    assert len(calls) == 2


def test_an_output_given_by_the_caller_counts_as_written(calls):
    """A graph that saved the tensor for its backward pass has to notice."""
    x, w, out = zeros(8, 16, dtype=torch.float32), zeros(16, 24, dtype=torch.float32), torch.ones(8, 24)
    leaf = torch.ones(8, 24, requires_grad=True)
    product = leaf * out                                   # saves out
    before = out._version
    with torch.no_grad():
        assert functional.linear(x, w, out=on_cuda(out)) is not None
    assert out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        functional.linear(x, w, out=on_cuda(torch.ones(8, 24)))     # (such tensors have no version)


def test_a_view_that_negates_its_memory_is_refused(calls):
    pair = torch.randn(16, 24, dtype=torch.complex64)
    x, w = zeros(8, 16, dtype=torch.float32), on_cuda(pair.conj().imag)
    assert w.is_neg()
    functional.linear(x, on_cuda(pair.imag))               # the same metadata otherwise
    with pytest.raises(ValueError, match="weight is a view that negates its memory"):
        functional.linear(x, w)
    functional.linear(x, on_cuda(pair.conj().imag.resolve_neg()))
    assert len(calls) == 2


@pytest.mark.parametrize("gate_rows", [True, False])
@pytest.mark.parametrize("up_rows", [True, False])
def test_gated_gradients_keep_the_layout_of_their_own_weight(calls, gate_rows, up_rows):
    M, K, N = 24, 40, 56
    weights = [zeros(K, N) if rows else zeros(N, K).t() for rows in (gate_rows, up_rows)]
    x, m = zeros(M, K), [zeros(M, N) for _ in range(3)]
    dx, *grads = functional.gated_linear_backward(m[0], x, *weights, m[1], m[2])
    assert dx.shape == x.shape
    for grad, weight in zip(grads, weights):
        assert grad.shape == weight.shape and grad.stride() == weight.stride()
    products = [c["name"] for c in calls[2:]]
    assert products == (["linear_pair_kernel"] if gate_rows == up_rows else ["linear_kernel"] * 2)


def test_threads_that_meet_at_a_first_call_load_its_kernel_once(calls, monkeypatch, no_leaks):
    """A second copy would stay loaded with nobody to release it."""
    import threading
    import time

    from triton_metal import kernels
    made, ready = [], threading.Barrier(4)

    class Slow(kernels.Linear):
        def __init__(self, *a):
            time.sleep(0.05)
            super().__init__(*a)
            made.append(self)

    monkeypatch.setattr(kernels, "Linear", Slow)
    x, w, failed = zeros(8, 16), zeros(16, 24), []

    def work():
        ready.wait()
        try:
            functional.linear(x, w)
        except Exception as e:      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and len(made) == 1 and len(calls) == 4
    functional.release()


def test_a_release_during_a_first_call_leaves_no_dead_recipe(calls, monkeypatch):
    """Another thread's release() between the load of a call's kernel and the call's end: later calls load it again."""
    real = functional._kernel
    monkeypatch.setattr(functional, "_kernel", lambda *a: (real(*a), functional.release())[0])
    x, w = zeros(8, 16), zeros(16, 24)
    with pytest.raises(StopIteration):          # (the launch that is written down finds no such kernel)
        functional.linear(x, w)
    monkeypatch.setattr(functional, "_kernel", real)
    functional.linear(x, w)
    assert len(calls) == 1


def test_statistics_of_rows_without_columns_are_refused(calls):
    """Nothing would be launched, and the statistics would be whatever their memory holds."""
    r, w = zeros(3, 0), zeros(0)
    total, normed = functional.residual_norm(r, r, w)
    assert total.shape == normed.shape == (3, 0)
    with pytest.raises(ValueError, match="rows without columns have no statistics"):
        functional.residual_norm(r, r, w, stats=True)
    functional.residual_norm(zeros(0, 8), None, zeros(8), stats=True)
