"""Host logic of the feed-forward kernels: IR and descriptors, argument names, and every refusal of
tmx_launch_on that needs no device.  The addresses here are made up; nothing is dereferenced, since a
launch that passes all checks ends at the missing device (or, where there is one, at the check that
the address is its memory)."""

import ctypes

import pytest

from triton_metal import _core, cuda, kernels

X, W, OUT, OTHER = 0x10000000, 0x20000000, 0x30000000, 0x40000000
BIG = 1 << 26


@pytest.fixture()
def load(no_leaks):
    made = []

    def make(cls, *args, **kw):
        made.append(cls(*args, **kw))
        return made[-1]

    yield make
    for kern in made:
        kern.release()


def launch(kern, pointers, lengths, scalars, stream=0):
    kern.launch_tensors(stream, pointers, lengths, scalars)


def refused(match, kern, pointers, lengths, scalars):
    with pytest.raises(RuntimeError, match=match):
        launch(kern, pointers, lengths, scalars)


NO_DEVICE = "no CUDA device|is not memory of device"


def linear_scalars(M, N, K, xm=None, xk=1, wk=None, wn=1, om=None, rm=None, pm=None):
    dense = lambda v, d: d if v is None else v  # noqa: E731
    return (M, N, K, dense(xm, K), xk, dense(wk, N), wn, dense(om, N), dense(rm, N), dense(pm, N))


def test_descriptor_round_trip_keeps_activation_and_norm(load):
    kern = load(kernels.Linear, "bf16", ("bias", "residual", "pre"), "gelu_tanh")
    assert "activation gelu_tanh" in kern.descriptor
    names = [line.split()[-1] for line in kern.descriptor.splitlines() if line.strip().startswith("arg")]
    assert names == list(kern.names)
    again = _core.compile_msl(kern.descriptor)
    _core.release_library(again)
    assert "norm layer" in load(kernels.ResidualNorm, "f32", (), None, "layer").descriptor
    assert "norm" not in load(kernels.ResidualNorm, "f32", (), None, "rms").descriptor.replace("residual_norm", "").replace(
        "normed", "")


@pytest.mark.parametrize("cls,operands", [
    (kernels.Linear, ("bias", "residual", "pre")), (kernels.GatedLinear, ("pre_gate", "pre_up")),
    (kernels.LinearSum, ()), (kernels.LinearPair, ()), (kernels.ActivationBackward, ("pre", "dz", "dbias")),
    (kernels.GatedActivationBackward, ()),
    (kernels.ResidualNorm, ("block", "bias", "gate", "post_weight", "sum", "stats")),
    (kernels.ResidualNormBackward, ("dsum", "block", "gate", "post_weight", "dresidual", "dblock", "dweight", "dbias",
                                    "dgate", "dpost_weight"))])
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_every_kernel_loads_with_and_without_its_optional_operands(load, cls, operands, element):
    assert len(load(cls, element, operands).metal_args) == len(cls.REQUIRED) + len(operands) + len(cls.SCALARS)
    load(cls, element)


@pytest.mark.parametrize("ir,match", [
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "M", "N", "K"), activation="swish", product=True),
     "activation 'swish'"),
    (kernels.feed_forward_ir("linear_sum_kernel", ("x", "w", "x2", "w2", "out", "M", "N", "K"), activation="relu",
                             product=True), "activation 'relu'"),
    (kernels.feed_forward_ir("residual_norm_kernel", ("residual", "weight", "normed", "scale", "eps", "M", "D"),
                             norm="batch"), "norm 'batch'"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "M", "N", "K")), "not the computation"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "M", "N"), product=True), "missing a required argument"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "out", "M", "N", "K"), product=True), "unknown or repeated"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "out2", "M", "N", "K"), product=True),
     "takes no argument 'out2'"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "M", "N", "K"), product=True).replace(
        "%w: !tt.ptr<bf16>", "%w: !tt.ptr<f16>"), "share one element type"),
    (kernels.feed_forward_ir("linear_kernel", ("x", "w", "out", "M", "N", "K"), product=True).replace("%M: i64", "%M: f32"),
     "unsupported type"),
    (kernels.feed_forward_ir("residual_norm_kernel", ("residual", "weight", "normed", "stats", "scale", "eps", "M", "D"))
     .replace("%stats: !tt.ptr<f32>", "%stats: !tt.ptr<bf16>"), "unsupported type"),
])
def test_modules_that_are_refused(ir, match):
    with pytest.raises(RuntimeError, match=match):
        _core.emit_msl(ir, 4)


def test_descriptors_that_are_refused(load):
    text = load(kernels.Linear, "bf16", (), "relu").descriptor
    for bad in (text.replace("activation relu", "activation swish"), text.replace("activation relu", "norm layer"),
                text.replace("pointer bf16 2 w", "pointer f16 2 w")):
        with pytest.raises(RuntimeError, match="MSL compilation failed"):
            _core.compile_msl(bad)


def test_options(load):
    kern, norm = load(kernels.Linear), load(kernels.ResidualNorm)
    cuda.set_option(kern.handle, "activation", 4)
    cuda.set_option(norm.handle, "layer_norm", 1)
    for handle, name, value in ((kern.handle, "activation", 6), (kern.handle, "activation", -1),
                                (norm.handle, "activation", 1), (kern.handle, "layer_norm", 1),
                                (kern.handle, "causal", 1), (load(kernels.LinearSum).handle, "activation", 1)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            cuda.set_option(handle, name, value)


def test_python_argument_names(load):
    kern = load(kernels.Linear, "f32", ("bias",))
    with pytest.raises(TypeError, match="missing 'bias'"):
        kern.arguments(x=1, w=2, out=3, M=1, N=1, K=1)
    with pytest.raises(TypeError, match="no argument 'pre'"):
        kern.arguments(x=1, w=2, out=3, bias=4, pre=5, M=1, N=1, K=1)
    with pytest.raises(TypeError, match="takes no operand"):
        kernels.Linear("f32", ("gate",))
    with pytest.raises(ValueError, match="unknown activation"):
        kernels.Linear("f32", (), "swish")
    with pytest.raises(ValueError, match="unknown norm"):
        kernels.ResidualNorm("f32", (), None, "batch")
    grid, kinds, values = kern.arguments(x=1, w=2, out=3, bias=4, M=300, N=200, K=7)
    assert grid == (3, 2, 1) and values[:4] == [1, 2, 3, 4] and values[4:] == [300, 200, 7, 7, 1, 200, 1, 200, 200, 200]


def test_linear_extents_and_strides(load):
    kern = load(kernels.Linear, "bf16")
    M, N, K = 8, 16, 32
    ok = [X, W, OUT], [M * K * 2, K * N * 2, M * N * 2]
    refused(NO_DEVICE, kern, *ok, linear_scalars(M, N, K))
    for i, name in enumerate(("x", "w", "out")):
        short = list(ok[1])
        short[i] -= 1
        refused(f"bytes of {name}, beyond", kern, ok[0], short, linear_scalars(M, N, K))
    refused("must not be negative", kern, *ok, linear_scalars(-1, N, K))
    refused("must not be negative", kern, *ok, linear_scalars(M, N, K, xm=-4))
    refused("above 2\\^31", kern, *ok, linear_scalars(1 << 31, N, K))
    refused("beyond its", kern, *ok, linear_scalars(M, N, K, xm=1 << 62))
    refused("rows of out overlap", kern, [X, W, OUT], [BIG] * 3, linear_scalars(M, N, K, om=N - 1))
    refused("not aligned", kern, [X + 1, W, OUT], [BIG] * 3, linear_scalars(M, N, K))
    refused("no valid address", kern, [X, 0, OUT], [BIG] * 3, linear_scalars(M, N, K))
    refused("no valid address", kern, [X, W, OUT], [BIG, -1, BIG], linear_scalars(M, N, K))
    # a stride of zero is a broadcast input and fine
    refused(NO_DEVICE, kern, [X, W, OUT], [K * 2, K * N * 2, M * N * 2], linear_scalars(M, N, K, xm=0))


def test_nothing_to_compute_needs_no_memory(load):
    for scalars in (linear_scalars(0, 16, 32), linear_scalars(8, 0, 32)):
        kern = load(kernels.Linear, "f16")
        try:
            launch(kern, [0, 0, 0], [0, 0, 0], scalars)
        except RuntimeError as e:
            assert "no CUDA device" in str(e)


def test_linear_aliasing(load):
    M, N, K = 64, 64, 64
    size = M * N * 2
    kern = load(kernels.Linear, "bf16", ("residual",))
    refused("out overlaps its input x", kern, [X, W, X, OTHER], [size] * 4, linear_scalars(M, N, K))
    refused("out overlaps its input x", kern, [X, W, X + size - 2, OTHER], [BIG] * 4, linear_scalars(M, N, K))
    refused("out overlaps its input w", kern, [X, W, W + 128, OTHER], [BIG] * 4, linear_scalars(M, N, K))
    refused(NO_DEVICE, kern, [X, W, OUT, OUT], [BIG] * 4, linear_scalars(M, N, K))             # in place
    refused("out overlaps its input residual", kern, [X, W, OUT, OUT + 2], [BIG] * 4, linear_scalars(M, N, K))
    refused("out overlaps its input residual", kern, [X, W, OUT, OUT], [BIG] * 4, linear_scalars(M, N, K, rm=N + 8))
    # side by side in one wider tensor
    refused(NO_DEVICE, kern, [X, W, OUT, OUT + N * 2], [BIG] * 4, linear_scalars(M, N, K, om=2 * N, rm=2 * N))
    refused("overlaps", kern, [X, W, OUT, OUT + N * 2 - 2], [BIG] * 4, linear_scalars(M, N, K, om=2 * N, rm=2 * N))
    pair = load(kernels.LinearPair, "bf16")
    refused("out and out2 overlap", pair, [X, W, X, W, OUT, OUT + 64], [BIG] * 6, (M, N, K, K, 1, N, 1, N))
    refused(NO_DEVICE, pair, [X, W, X, W, OUT, OTHER], [BIG] * 6, (M, N, K, K, 1, N, 1, N))


def test_activation_bwd_refusals(load):
    kern = load(kernels.ActivationBackward, "f16", ("dz",), "gelu")
    refused("needs the pre-activations", kern, [X, OUT], [BIG] * 2, (8, 8, 8, 8, 8))
    kern = load(kernels.ActivationBackward, "f16", ("pre", "dz"), "gelu")
    refused(NO_DEVICE, kern, [X, W, X], [BIG] * 3, (8, 8, 8, 8, 8))
    refused("overlaps its input dout", kern, [X, W, X + 16], [BIG] * 3, (8, 8, 8, 8, 8))
    gated = load(kernels.GatedActivationBackward, "f16", (), "silu")
    refused("dgate and dup overlap", gated, [X, W, OTHER, OUT, OUT], [BIG] * 5, (8, 8, 8, 8, 8))
    refused(NO_DEVICE, gated, [X, W, OTHER, W, OTHER], [BIG] * 5, (8, 8, 8, 8, 8))


def test_norm_refusals(load):
    one, eps = _core.float_bits(1.0), _core.float_bits(1e-6)
    kern = load(kernels.ResidualNorm, "f32")
    refused("at most 16384 columns", kern, [X, W, OUT], [BIG] * 3, (1, 16385, one, eps, 16385))
    refused("eps must not be negative", kern, [X, W, OUT], [BIG] * 3, (1, 16, one, _core.float_bits(-1.0), 16))
    refused("eps must not be negative", kern, [X, W, OUT], [BIG] * 3, (1, 16, one, _core.float_bits(float("nan")), 16))
    refused(NO_DEVICE, kern, [X, W, X], [BIG] * 3, (4, 16, one, eps, 16))
    refused("rows of normed overlap", kern, [X, W, OUT], [BIG] * 3, (4, 16, one, eps, 8))
    refused("needs the block's output", load(kernels.ResidualNorm, "f32", ("gate",)), [X, W, OUT, OTHER], [BIG] * 4,
            (4, 16, one, eps, 16))
    stats = load(kernels.ResidualNorm, "f32", ("stats",))
    refused("aligned to 16", stats, [X, W, OUT, OTHER + 4], [BIG] * 4, (4, 16, one, eps, 16))
    refused("stats overlaps normed", stats, [X, W, OUT, OUT + 16], [BIG] * 4, (4, 16, one, eps, 16))
    refused("bytes of stats", stats, [X, W, OUT, OTHER], [BIG] * 3 + [63], (4, 16, one, eps, 16))
    bwd = load(kernels.ResidualNormBackward, "f32", ("dgate",))
    refused("not there", bwd, [X, W, OTHER, OUT, OUT + BIG], [BIG] * 5, (4, 16, one, 16))
    bwd = load(kernels.ResidualNormBackward, "f32", ("dsum", "dresidual", "dweight"))
    refused(NO_DEVICE, bwd, [X, W, OTHER, OUT, OUT + BIG, OUT + BIG, X + BIG], [BIG] * 7, (4, 16, one, 16))
    refused("dresidual overlaps its input sum", bwd, [X, W, OTHER, OUT, OUT + BIG, W, X + BIG], [BIG] * 7,
            (4, 16, one, 16))


def test_launch_on_refusals(load):
    kern = load(kernels.Linear, "bf16")
    kinds, values = kern._kinds, kern._values(X, W, OUT, *linear_scalars(1, 1, 1))
    lengths = kern._values(*([BIG] * len(kern.names)))
    call = cuda._lib.tmx_launch_on

    def bad(match, *args):
        assert call(*args) == -1
        assert match in _core.last_error()

    bad("is not live", 1 << 40, 0, 1, 1, 1, 128, kinds, values, lengths, len(kinds))
    bad("no lengths", kern.handle, 0, 1, 1, 1, 128, kinds, values, None, len(kinds))
    bad("NULL argument arrays", kern.handle, 0, 1, 1, 1, 128, None, values, lengths, len(kinds))
    bad("arguments", kern.handle, 0, 1, 1, 1, 128, kinds, values, lengths, len(kinds) - 1)
    bad("grid must be positive", kern.handle, 0, 0, 1, 1, 128, kinds, values, lengths, len(kinds))
    bad("threadsPerThreadgroup", kern.handle, 0, 1, 1, 1, 2048, kinds, values, lengths, len(kinds))
    wrong = (ctypes.c_int32 * len(kinds))(*kinds)
    wrong[0] = 5
    bad("kind 5", kern.handle, 0, 1, 1, 1, 128, wrong, values, lengths, len(kinds))
    wrong[0] = 1
    bad("is a pointer", kern.handle, 0, 1, 1, 1, 128, wrong, values, lengths, len(kinds))
    mm = load(kernels.Matmul, "bf16")
    bad("takes the feed-forward kernels", mm.handle, 0, 1, 1, 1, 128, kinds, values, lengths, len(kinds))
    # tm_launch itself takes no raw addresses
    with pytest.raises(RuntimeError, match="unknown launch argument kind 4"):
        _core.launch(kern.handle, (1, 1, 1), 128, [4] * len(kinds), [0] * len(kinds))
