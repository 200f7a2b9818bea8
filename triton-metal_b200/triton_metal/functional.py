"""The feed-forward operators on torch tensors.

    linear            out = act(x @ weight + bias) + residual
    gated_linear      h = act(x @ w_gate) * (x @ w_up)
    residual_norm     sum = scale * residual + gate * post(block), normed = norm(sum) * weight + bias

and their backward passes, each one or a few launches of this library's kernels (kernels.Linear,
GatedLinear, ..., through tmx_launch_on) on torch's current stream.  Nothing waits, nothing is
cached between calls but the loaded kernels, and a call may be captured into a CUDA graph.  All
tensors live on the library's device and share one element type: float32, float16 or bfloat16.

x may have leading dimensions ([..., K]); weights are [K, N] with either dimension contiguous, so a
weight stored [N, K] is passed as its transposed view.  Gradients are explicit functions: they take
what the forward pass returned and return contiguous tensors (a weight's gradient in the layout of
the weight).  The reference has no counterpart.
"""

import math

import torch

from . import _core, cuda, kernels

_ELEMENT = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
_loaded = {}


def _kernel(cls, dtype, operands, activation=None, norm=None):
    key = (cls, dtype, operands, activation, norm)
    kern = _loaded.get(key)
    if kern is None:
        kern = _loaded[key] = cls(_ELEMENT[dtype], operands, activation, norm)
    return kern


def release():
    """Drop the loaded kernels (they are loaded again on the next call)."""
    for kern in _loaded.values():
        kern.release()
    _loaded.clear()


def _check(name, t, dtype, device, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, the other operands are {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands are on {device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    return t


def _first(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype not in _ELEMENT:
        raise TypeError(f"{name} is {t.dtype}; float32, float16 and bfloat16 are supported")
    if not t.is_cuda or t.device.index != cuda.get_device():
        raise ValueError(f"{name} is on {t.device}; this process's device is cuda:{cuda.get_device()}")
    if t.dim() < 1:
        raise ValueError(f"{name} needs at least one dimension")
    return t.dtype, t.device


def _rows(name, t):
    """[..., C] as [R, C] with unit column stride (a copy only where no view has that form)."""
    t = t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _strides(t):
    """Both strides of a matrix; those of dimensions of one element are made the dense ones."""
    a, b = t.stride()
    rows, cols = t.shape
    if cols <= 1 and rows <= 1:
        return max(cols, 1), 1
    if cols <= 1:
        b = 1
    if rows <= 1:
        a = max(cols, 1) if b == 1 else 1
    return a, b


def _vector(name, t, dtype, device, n):
    if t is None:
        return None
    _check(name, t, dtype, device, (n,))
    return t if t.stride(0) == 1 or n <= 1 else t.contiguous()


def _launch(kern, tensors, scalars, device):
    pointers, lengths = [], []
    for t in tensors:
        pointers.append(t.data_ptr())
        # (an empty view has no address, whatever its storage holds)
        lengths.append(t.untyped_storage().nbytes() - t.storage_offset() * t.element_size() if t.numel() else 0)
    kern.launch_tensors(torch.cuda.current_stream(device).cuda_stream, pointers, lengths, scalars)


def _weight(name, w, dtype, device, K):
    _check(name, w, dtype, device)
    if w.dim() != 2 or w.shape[0] != K:
        raise ValueError(f"{name} has shape {tuple(w.shape)}, expected ({K}, N)")
    return w


def _activation(name):
    if name not in cuda.ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}; expected one of {', '.join(cuda.ACTIVATIONS)}")
    return name


def linear(x, weight, bias=None, residual=None, activation="none", *, pre=False, out=None):
    """act(x @ weight + bias) + residual; with pre=True also x @ weight + bias, which the backward
    pass of an activation reads.  `out` may be `residual` itself."""
    dtype, device = _first("x", x)
    _activation(activation)
    x2 = _rows("x", x)
    M, K = x2.shape
    _weight("weight", weight, dtype, device, K)
    N = weight.shape[1]
    shape = x.shape[:-1] + (N,)
    bias = _vector("bias", bias, dtype, device, N)
    if residual is not None:
        _check("residual", residual, dtype, device, tuple(shape))
        r2 = _rows("residual", residual)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
    else:
        _check("out", out, dtype, device, tuple(shape))
        if out.numel() and not (out.dim() == 2 and (out.stride(1) == 1 or N <= 1)) and not out.is_contiguous():
            raise ValueError("out must be contiguous, or a matrix with contiguous rows")
    o2 = out if out.dim() == 2 else out.view(M, N)
    z = torch.empty(shape, dtype=dtype, device=device) if pre else None
    tensors, operands = [x2, weight, o2], ()
    if bias is not None:
        tensors.append(bias)
        operands += ("bias",)
    if residual is not None:
        tensors.append(r2)
        operands += ("residual",)
    if pre:
        tensors.append(z)
        operands += ("pre",)
    _launch(_kernel(kernels.Linear, dtype, operands, activation), tensors,
            (M, N, K, *_strides(x2), *_strides(weight), _row_stride(o2),
             _row_stride(r2) if residual is not None else N, N), device)
    return (out, z) if pre else out


def _product(a, b, device, out=None):
    """a @ b of matrices with any strides."""
    M, K = a.shape
    N = b.shape[1]
    out = torch.empty((M, N), dtype=a.dtype, device=device) if out is None else out
    _launch(_kernel(kernels.Linear, a.dtype, ()), (a, b, out),
            (M, N, K, *_strides(a), *_strides(b), _row_stride(out), N, N), device)
    return out


def _by_columns(w):
    """Whether a [K, N] weight is stored [N, K]."""
    return w.stride(0) == 1 and w.stride(1) != 1


def linear_backward(dout, x, weight, pre=None, activation="none", *, bias=False):
    """(dx, dweight, dbias or None) of linear; the gradient of the residual is dout itself.  `pre` is
    what linear returned with pre=True (not needed without an activation)."""
    dtype, device = _first("dout", dout)
    _activation(activation)
    x2 = _rows("x", _check("x", x, dtype, device))
    M, K = x2.shape
    _weight("weight", weight, dtype, device, K)
    N = weight.shape[1]
    _check("dout", dout, dtype, device, tuple(x.shape[:-1]) + (N,))
    d2 = _rows("dout", dout)
    if activation != "none":
        if pre is None:
            raise ValueError(f"the backward pass of {activation} needs the pre-activations")
        p2 = _rows("pre", _check("pre", pre, dtype, device, tuple(dout.shape)))
    db = torch.empty(N, dtype=dtype, device=device) if bias else None
    dz = d2
    if activation != "none" or bias:
        tensors, operands = [d2], ()
        if activation != "none":
            dz = torch.empty((M, N), dtype=dtype, device=device)
            tensors += [p2, dz]
            operands += ("pre", "dz")
        if bias:
            tensors.append(db)
            operands += ("dbias",)
        _launch(_kernel(kernels.ActivationBackward, dtype, operands, activation), tensors,
                (M, N, _row_stride(d2), _row_stride(p2) if activation != "none" else N, N), device)
    dx = _product(dz, weight.t(), device).view(x.shape)
    if _by_columns(weight):
        dw = _product(dz.t(), x2, device).t()
    else:
        dw = _product(x2.t(), dz, device)
    return dx, dw, db


def gated_linear(x, w_gate, w_up, activation="silu", *, save=False):
    """act(x @ w_gate) * (x @ w_up); with save=True also the two products, for the backward pass."""
    dtype, device = _first("x", x)
    _activation(activation)
    x2 = _rows("x", x)
    M, K = x2.shape
    _weight("w_gate", w_gate, dtype, device, K)
    N = w_gate.shape[1]
    _check("w_up", w_up, dtype, device, (K, N))
    if _strides(w_up) != _strides(w_gate):
        w_up = _like(w_up, w_gate)
    shape = x.shape[:-1] + (N,)
    h = torch.empty(shape, dtype=dtype, device=device)
    if save:
        g, u = torch.empty_like(h), torch.empty_like(h)
    _launch(_kernel(kernels.GatedLinear, dtype, ("pre_gate", "pre_up") if save else (), activation),
            (x2, w_gate, w_up, h, g, u) if save else (x2, w_gate, w_up, h),
            (M, N, K, *_strides(x2), *_strides(w_gate), N, N), device)
    return (h, g, u) if save else h


def _like(t, other):
    """A copy of t with the strides of other."""
    copy = torch.empty_strided(other.shape, other.stride(), dtype=t.dtype, device=t.device)
    copy.copy_(t)
    return copy


def gated_linear_backward(dh, x, w_gate, w_up, pre_gate, pre_up, activation="silu"):
    """(dx, dw_gate, dw_up) of gated_linear, from the products it saved."""
    dtype, device = _first("dh", dh)
    _activation(activation)
    x2 = _rows("x", _check("x", x, dtype, device))
    M, K = x2.shape
    _weight("w_gate", w_gate, dtype, device, K)
    N = w_gate.shape[1]
    _check("w_up", w_up, dtype, device, (K, N))
    if _strides(w_up) != _strides(w_gate):
        w_up = _like(w_up, w_gate)
    _check("dh", dh, dtype, device, tuple(x.shape[:-1]) + (N,))
    d2 = _rows("dh", dh)
    g2 = _rows("pre_gate", _check("pre_gate", pre_gate, dtype, device, tuple(dh.shape)))
    u2 = _rows("pre_up", _check("pre_up", pre_up, dtype, device, tuple(dh.shape)))
    if _row_stride(g2) != _row_stride(u2):
        g2, u2 = g2.contiguous(), u2.contiguous()
    both = torch.empty((2, M, N), dtype=dtype, device=device)
    dg, du = both[0], both[1]
    _launch(_kernel(kernels.GatedActivationBackward, dtype, (), activation), (d2, g2, u2, dg, du),
            (M, N, _row_stride(d2), _row_stride(g2), N), device)
    wg, wu = w_gate.t(), w_up.t()
    dx = torch.empty((M, K), dtype=dtype, device=device)
    _launch(_kernel(kernels.LinearSum, dtype, ()), (dg, wg, du, wu, dx),
            (M, K, N, *_strides(dg), *_strides(wg), max(K, 1)), device)
    if _by_columns(w_gate):
        dwg, dwu = (torch.empty((N, K), dtype=dtype, device=device) for _ in range(2))
        a, b = dg.t(), du.t()
        _launch(_kernel(kernels.LinearPair, dtype, ()), (a, x2, b, x2, dwg, dwu),
                (N, K, M, *_strides(a), *_strides(x2), max(K, 1)), device)
        dwg, dwu = dwg.t(), dwu.t()
    else:
        dwg, dwu = (torch.empty((K, N), dtype=dtype, device=device) for _ in range(2))
        a = x2.t()
        _launch(_kernel(kernels.LinearPair, dtype, ()), (a, dg, a, du, dwg, dwu),
                (K, N, M, *_strides(a), *_strides(dg), max(N, 1)), device)
    return dx.view(x.shape), dwg, dwu


def _same_rows(tensors):
    """Matrices with one row stride: contiguous copies of those that differ from dense rows, unless all agree."""
    present = [t for t in tensors if t is not None]
    first = _row_stride(present[0])
    if all(_row_stride(t) == first for t in present):
        return tensors, first
    return [t if t is None else t.contiguous() for t in tensors], max(present[0].shape[1], 1)


def _norm_kind(kind):
    if kind not in ("rms", "layer"):
        raise ValueError(f"unknown norm {kind!r}; expected 'rms' or 'layer'")
    return kind


def residual_norm(residual, block=None, weight=None, bias=None, gate=None, post_weight=None, *, kind="rms", scale=1.0,
                  eps=1e-6, stats=False):
    """(sum, normed), or (sum, normed, stats) with stats=True:

        t = norm(block) * post_weight, or block;  sum = scale * residual + gate * t
        normed = norm(sum) * weight + bias

    Without a block (and with scale 1) sum is residual itself.  stats, [rows, 4] float32, is what the
    backward pass reads: mean and 1/deviation of each row of sum, then of block."""
    dtype, device = _first("residual", residual)
    _norm_kind(kind)
    D = residual.shape[-1]
    if weight is None:
        raise ValueError("residual_norm needs the norm's weight")
    weight = _vector("weight", weight, dtype, device, D)
    bias = _vector("bias", bias, dtype, device, D)
    gate = _vector("gate", gate, dtype, device, D)
    post_weight = _vector("post_weight", post_weight, dtype, device, D)
    if block is None and (gate is not None or post_weight is not None):
        raise ValueError("a gate or a norm behind the block needs the block's output")
    r2 = _rows("residual", residual)
    M = r2.shape[0]
    shape = residual.shape
    y2 = None if block is None else _rows("block", _check("block", block, dtype, device, tuple(shape)))
    # the results are dense, and one row stride holds for all
    r2 = r2 if _row_stride(r2) == max(D, 1) else r2.contiguous()
    y2 = y2 if y2 is None or _row_stride(y2) == max(D, 1) else y2.contiguous()
    normed = torch.empty(shape, dtype=dtype, device=device)
    total = residual if block is None and scale == 1.0 else torch.empty(shape, dtype=dtype, device=device)
    tensors, operands = [r2, weight, normed], ()
    rows = torch.empty((M, 4), dtype=torch.float32, device=device) if stats else None
    for name, t in (("block", y2), ("bias", bias), ("gate", gate), ("post_weight", post_weight),
                    ("sum", None if total is residual else total), ("stats", rows)):
        if t is not None:
            tensors.append(t)
            operands += (name,)
    _launch(_kernel(kernels.ResidualNorm, dtype, operands, None, kind), tensors,
            (M, D, _core.float_bits(scale), _core.float_bits(eps), max(D, 1)), device)
    return (total, normed, rows) if stats else (total, normed)


def residual_norm_backward(dnormed, dsum, total, stats, weight, block=None, gate=None, post_weight=None, *, kind="rms",
                           scale=1.0, bias=False):
    """(dresidual, dblock, dweight, dbias, dgate, dpost_weight) of residual_norm, None where the operand
    was not there.  dsum, the gradient that reaches sum past the norm, may be None."""
    dtype, device = _first("dnormed", dnormed)
    _norm_kind(kind)
    D = dnormed.shape[-1]
    shape = tuple(dnormed.shape)
    weight = _vector("weight", weight, dtype, device, D)
    gate = _vector("gate", gate, dtype, device, D)
    post_weight = _vector("post_weight", post_weight, dtype, device, D)
    if block is None and (gate is not None or post_weight is not None):
        raise ValueError("a gate or a norm behind the block needs the block's output")
    dn = _rows("dnormed", dnormed)
    M = dn.shape[0]
    _check("stats", stats, torch.float32, device, (M, 4))
    s2 = _rows("sum", _check("sum", total, dtype, device, shape))
    ds = None if dsum is None else _rows("dsum", _check("dsum", dsum, dtype, device, shape))
    y2 = None if block is None else _rows("block", _check("block", block, dtype, device, shape))
    dense = max(D, 1)
    dn, s2, ds, y2 = (t if t is None or _row_stride(t) == dense else t.contiguous() for t in (dn, s2, ds, y2))
    stats = stats.contiguous()
    empty = lambda *size: torch.empty(size, dtype=dtype, device=device)  # noqa: E731
    dresidual, dweight = empty(*shape), empty(D)
    dblock = empty(*shape) if block is not None else None
    dbias = empty(D) if bias else None
    dgate = empty(D) if gate is not None else None
    dpost = empty(D) if post_weight is not None else None
    tensors, operands = [dn, s2, stats, weight], ()
    for name, t in (("dsum", ds), ("block", y2), ("gate", gate), ("post_weight", post_weight),
                    ("dresidual", dresidual), ("dblock", dblock), ("dweight", dweight), ("dbias", dbias),
                    ("dgate", dgate), ("dpost_weight", dpost)):
        if t is not None:
            tensors.append(t)
            operands += (name,)
    _launch(_kernel(kernels.ResidualNormBackward, dtype, operands, None, kind), tensors,
            (M, D, _core.float_bits(scale), dense), device)
    return dresidual, dblock, dweight, dbias, dgate, dpost
