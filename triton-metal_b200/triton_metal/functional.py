"""The feed-forward operators on torch tensors.

    linear            out = act(x @ weight + bias) + residual
    gated_linear      h = act(x @ w_gate) * (x @ w_up)
    residual_norm     sum = scale * residual + gate * post(block), normed = norm(sum) * weight + bias

and their backward passes, each one or a few launches of this library's kernels (kernels.Linear,
GatedLinear, ..., through tmx_launch_on) on torch's current stream.  Nothing waits, and a call may be
captured into a CUDA graph.  All tensors live on the library's device and share one element type:
float32, float16 or bfloat16.

x may have leading dimensions ([..., K]); weights are [K, N] with either dimension contiguous, so a
weight stored [N, K] is passed as its transposed view.  Gradients are explicit functions: they take
what the forward pass returned and return new tensors (a weight's gradient in the layout of the
weight).  No graph is recorded, so an operand that requires grad is refused while grad mode is on (and one
that carries a forward-mode tangent always).  The reference has no counterpart.

Operands that the kernels cannot take as they lie are copied on every call: an x whose leading dimensions are
not a fixed distance apart or whose rows are not contiguous, a vector with a stride, [rows, D] operands of the
norms that are not dense (a column slice of a wider tensor), one of two gate and up weights in different
layouts, and, inside the library, 16-bit operands of a product that are not aligned to 16 bytes.

Every call goes through a recipe: the checks of shapes, types and strides, the temporaries, and the
launches with everything but the addresses.  Recipes depend on the operands' metadata alone and are
kept by it, so a repeated call pays for its allocations, its addresses and its launches; the library
checks addresses (device, alignment, overlap) on every launch.
"""

import math
import struct
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _core, cuda, kernels

_ELEMENT = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
_KERNELS = {}
_RECIPES = {}
_MOST_RECIPES = 4096
_loading = threading.Lock()
_released = [0]             # how often release() has run
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def release():
    """Drop the loaded kernels and recipes (they are made again on the next call)."""
    with _loading:
        _released[0] += 1
        _RECIPES.clear()
        while _KERNELS:
            _KERNELS.popitem()[1].release()


def check():
    """Raise if a kernel among the work that has finished gave up a wait: its results are not valid.

    The kernels' waits are bounded.  One that runs out is reported by the next call of this module, which then
    launches nothing; a program whose last call it may have been, or that replays graphs, synchronises and asks
    here."""
    cuda.check_status()


def _kernel(cls, dtype, operands=(), activation=None, norm=None):
    key = (cls, dtype, operands, activation, norm)
    kern = _KERNELS.get(key)
    if kern is None:
        with _loading:                  # threads that meet here load it once
            kern = _KERNELS.get(key)
            if kern is None:
                kern = _KERNELS[key] = cls(_ELEMENT[dtype], operands, activation, norm)
    return kern


class _Matrix:
    """Rows and columns with two strides, in the tensor at `slot` of a recipe."""
    __slots__ = ("slot", "rows", "cols", "s0", "s1")

    def __init__(self, slot, rows, cols, s0, s1):
        # strides of dimensions of one element are made the dense ones
        if cols <= 1:
            s1 = 1
        if rows <= 1:
            s0 = max(cols, 1) if s1 == 1 else 1
        self.slot, self.rows, self.cols, self.s0, self.s1 = slot, rows, cols, s0, s1

    @property
    def T(self):
        return _Matrix(self.slot, self.cols, self.rows, self.s1, self.s0)

    def span(self):
        return 0 if not self.rows or not self.cols else (self.rows - 1) * self.s0 + (self.cols - 1) * self.s1 + 1


class _Recipe:
    """`tensors`: the operands by name; what is None is left out."""

    def __init__(self, **tensors):
        first_name, first = next(iter(tensors.items()))
        for name, t in tensors.items():
            if t is not None and not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
        if first.dtype not in _ELEMENT:
            raise TypeError(f"{first_name} is {first.dtype}; float32, float16 and bfloat16 are supported")
        if not first.is_cuda or first.device.index != cuda.get_device():
            raise ValueError(f"{first_name} is on {first.device}; this process's device is cuda:{cuda.get_device()}")
        self.dtype, self.device, self.index = first.dtype, first.device, first.device.index
        self.width = first.element_size()
        for name, t in tensors.items():
            if t is None:
                continue
            expected = torch.float32 if name == "stats" else self.dtype
            if t.dtype != expected:
                raise TypeError(f"{name} is {t.dtype}, expected {expected}")
            if t.device != self.device:
                raise ValueError(f"{name} is on {t.device}, the other operands are on {self.device}")
            if t.requires_grad and _grad_enabled():
                raise RuntimeError(f"{name} requires grad" + _NO_GRAPH)
            if t.is_neg():
                raise ValueError(f"{name} is a view that negates its memory; pass {name}.resolve_neg()")
        self.tensors = tensors
        self.slots = {name: i for i, name in enumerate(tensors)}
        self.copies, self.allocs, self.steps, self.results = [], [], [], []

    # ---- operands -------------------------------------------------------------------------
    def shape(self, name, shape):
        t = self.tensors[name]
        if t is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")

    def rows(self, name, dense=False, writable=False):
        """[..., C] as a matrix with unit column stride: a view where there is one, else a copy."""
        t = self.tensors[name]
        if t is None:
            return None
        if t.dim() < 1:
            raise ValueError(f"{name} needs at least one dimension")
        rows, cols, slot = math.prod(t.shape[:-1]), t.shape[-1], self.slots[name]
        view = t if t.dim() == 2 else None
        if view is None:
            try:
                view = t.view(rows, cols)
            except RuntimeError:
                pass
        if view is not None and (view.stride(1) == 1 or cols <= 1):
            m = _Matrix(slot, rows, cols, *view.stride())
            if not dense or m.s0 == max(cols, 1):
                return m
        if writable:
            raise ValueError(f"{name} must have contiguous rows a fixed distance apart")
        self.copies.append((slot, (rows, cols)))
        return _Matrix(slot, rows, cols, max(cols, 1), 1)

    def matrix(self, name, rows, cols=None):
        t = self.tensors[name]
        if t.dim() != 2 or t.shape[0] != rows or (cols is not None and t.shape[1] != cols):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({rows}, {'N' if cols is None else cols})")
        return _Matrix(self.slots[name], t.shape[0], t.shape[1], *t.stride())

    def vector(self, name, n):
        t = self.tensors[name]
        if t is None:
            return None
        self.shape(name, (n,))
        if t.stride(0) != 1 and n > 1:
            self.copies.append((self.slots[name], (n,)))
        return _Matrix(self.slots[name], 1, n, max(n, 1), 1)

    def new(self, shape, dtype=None):
        """A new dense tensor, as a matrix of its rows."""
        slot = len(self.tensors) + len(self.allocs)
        self.allocs.append((tuple(shape), dtype or self.dtype))
        rows, cols = math.prod(shape[:-1]), shape[-1]
        return _Matrix(slot, rows, cols, max(cols, 1), 1)

    # ---- launches ---------------------------------------------------------------------------
    def launch(self, cls, operands, scalars, activation=None, norm=None):
        """`operands`: name -> matrix; None is left out.  `scalars` in the kernel's order."""
        present = {name: m for name, m in operands.items() if m is not None}
        kern = _kernel(cls, self.dtype, tuple(n for n in cls.OPTIONAL if n in present), activation, norm)
        slots = [present[n].slot for n in kern.pointers]
        n = len(kern.names)
        lengths = [present[n_].span() * (4 if n_ == "stats" else self.width) for n_ in kern.pointers]
        pack = struct.Struct(f"{len(slots)}q").pack
        numbers = struct.pack(f"{len(scalars)}q", *scalars)
        grid = kern._grid(scalars[0], scalars[1])
        self.steps.append((kern.handle, grid[0], grid[1], kern.threads, kern._kinds, slots, pack, numbers,
                           pack(*lengths) + bytes(len(numbers)), n))

    def product(self, x, w, out):
        self.launch(kernels.Linear, dict(x=x, w=w, out=out),
                    (x.rows, w.cols, x.cols, x.s0, x.s1, w.s0, w.s1, out.s0, out.s0, out.s0))

    def run(self, tensors):
        slots = list(tensors)
        for slot, shape in self.copies:
            slots[slot] = slots[slot].reshape(shape).contiguous()
        new = tensors[0].new_empty
        for shape, dtype in self.allocs:
            slots.append(new(shape) if dtype is self.dtype else new(shape, dtype=dtype))
        stream = _raw_stream(self.index) if _raw_stream else torch.cuda.current_stream(self.device).cuda_stream
        for handle, gx, gy, threads, kinds, used, pack, numbers, lengths, n in self.steps:
            if _launch_on(handle, stream, gx, gy, 1, threads, kinds, pack(*[slots[i].data_ptr() for i in used]) + numbers,
                          lengths, n):
                raise RuntimeError(_core.last_error())
        results = [None if r is None else slots[r[0]] if r[1] is None else r[1](slots[r[0]]) for r in self.results]
        return results[0] if len(results) == 1 else tuple(results)


_launch_on = cuda._lib.tmx_launch_on
_grad_enabled = torch.is_grad_enabled
_NO_GRAPH = (", and these functions record no graph: call them under torch.no_grad() (or on detached tensors) and take "
             "the gradients from the backward functions")


def _refuse_tangents(names, tensors):
    for name, t in zip(names, tensors):
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} carries a forward-mode tangent" + _NO_GRAPH)


def _keep(key, recipe, released):
    recipe.tensors = dict.fromkeys(recipe.tensors)       # metadata only: no operand is held
    with _loading:
        if released != _released[0]:                     # its kernels have been dropped since
            return
        if len(_RECIPES) >= _MOST_RECIPES:
            _RECIPES.clear()
        _RECIPES[key] = recipe


def _call(build, static, names, tensors):
    """Run the recipe for these operands, made by `build` on first sight of their metadata."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(names, tensors)
    try:
        key = (build, static, _grad_enabled(),
               tuple([None if t is None else (t.dtype, t.get_device(), t.shape, t.stride(), t.requires_grad, t.is_neg())
                      for t in tensors]))
        recipe = _RECIPES.get(key)
    except AttributeError:          # not a tensor: the recipe says which
        key = recipe = None
    if recipe is None:
        released = _released[0]
        recipe = _Recipe(**dict(zip(names, tensors)))
        build(recipe, *static)
        _keep(key, recipe, released)
    return recipe.run(tensors)


def _activation(name):
    if name not in cuda.ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}; expected one of {', '.join(cuda.ACTIVATIONS)}")


def _transposed(t):
    return t.t()


# ---- linear ------------------------------------------------------------------------------------

def _plan_linear(r, activation, pre):
    _activation(activation)
    x = r.rows("x")
    w = r.matrix("weight", x.cols)
    shape = tuple(r.tensors["x"].shape[:-1]) + (w.cols,)
    r.shape("residual", shape)
    r.shape("out", shape)
    bias, residual = r.vector("bias", w.cols), r.rows("residual")
    out = r.rows("out", writable=True) if r.tensors["out"] is not None else r.new(shape)
    z = r.new(shape) if pre else None
    r.launch(kernels.Linear, dict(x=x, w=w, out=out, bias=bias, residual=residual, pre=z),
             (x.rows, w.cols, x.cols, x.s0, x.s1, w.s0, w.s1, out.s0, residual.s0 if residual else out.s0,
              z.s0 if z else out.s0), activation)
    r.results = [(out.slot, None)] + ([(z.slot, None)] if pre else [])


def linear(x, weight, bias=None, residual=None, activation="none", *, pre=False, out=None):
    """act(x @ weight + bias) + residual; with pre=True also x @ weight + bias, which the backward
    pass of an activation reads.  `out` may be `residual` itself."""
    result = _call(_plan_linear, (activation, bool(pre)), ("x", "weight", "bias", "residual", "out"),
                   (x, weight, bias, residual, out))
    if out is not None and not out.is_inference():
        increment_version(out)          # a graph that saved it notices
    return result


def _weight_gradient(r, x, dz, weight):
    """The matrix and the result of x^T dz in the layout of the weight."""
    if weight.s0 == 1 and weight.s1 != 1:
        dw = r.new((weight.cols, weight.rows))
        return dw, (dz.T, x), (dw.slot, _transposed)
    dw = r.new((weight.rows, weight.cols))
    return dw, (x.T, dz), (dw.slot, None)


def _plan_linear_backward(r, activation, bias):
    _activation(activation)
    r.shape("x", tuple(r.tensors["dout"].shape[:-1]) + tuple(r.tensors["x"].shape[-1:]))
    x = r.rows("x")
    w = r.matrix("weight", x.cols)
    r.shape("dout", tuple(r.tensors["x"].shape[:-1]) + (w.cols,))
    dout = r.rows("dout")
    db = r.new((w.cols,)) if bias else None
    dz = dout
    if activation != "none":
        if r.tensors["pre"] is None:
            raise ValueError(f"the backward pass of {activation} needs the pre-activations")
        r.shape("pre", r.tensors["dout"].shape)
        pre = r.rows("pre")
        dz = r.new((dout.rows, w.cols))
        r.launch(kernels.ActivationBackward, dict(dout=dout, pre=pre, dz=dz, dbias=db),
                 (dout.rows, w.cols, dout.s0, pre.s0, dz.s0), activation)
    elif bias:
        r.launch(kernels.ActivationBackward, dict(dout=dout, dbias=db), (dout.rows, w.cols, dout.s0, dout.s0, dout.s0),
                 activation)
    dx = r.new(r.tensors["x"].shape)
    r.product(dz, w.T, dx)
    dw, (a, b), result = _weight_gradient(r, x, dz, w)
    r.product(a, b, dw)
    r.results = [(dx.slot, None), result, (db.slot, None) if bias else None]


def linear_backward(dout, x, weight, pre=None, activation="none", *, bias=False):
    """(dx, dweight, dbias or None) of linear; the gradient of the residual is dout itself.  `pre` is
    what linear returned with pre=True (not needed without an activation)."""
    return _call(_plan_linear_backward, (activation, bool(bias)), ("dout", "x", "weight", "pre"),
                 (dout, x, weight, None if activation == "none" else pre))


# ---- gated linear ---------------------------------------------------------------------------------

def _gated_weights(r, K):
    """Both weights with the strides of w_gate."""
    wg = r.matrix("w_gate", K)
    wu = r.matrix("w_up", K, wg.cols)
    if (wg.s0, wg.s1) == (wu.s0, wu.s1):
        return wg, wu
    # one of the two is copied into the layout of the other: the one that is not dense rows
    if (wg.s0, wg.s1) != (max(wg.cols, 1), 1):
        r.copies.append((wg.slot, (wg.rows, wg.cols)))
    if (wu.s0, wu.s1) != (max(wu.cols, 1), 1):
        r.copies.append((wu.slot, (wu.rows, wu.cols)))
    return (_Matrix(m.slot, m.rows, m.cols, max(m.cols, 1), 1) for m in (wg, wu))


def _plan_gated_linear(r, activation, save):
    _activation(activation)
    x = r.rows("x")
    wg, wu = _gated_weights(r, x.cols)
    shape = tuple(r.tensors["x"].shape[:-1]) + (wg.cols,)
    h = r.new(shape)
    g, u = (r.new(shape), r.new(shape)) if save else (None, None)
    r.launch(kernels.GatedLinear, dict(x=x, w_gate=wg, w_up=wu, out=h, pre_gate=g, pre_up=u),
             (x.rows, wg.cols, x.cols, x.s0, x.s1, wg.s0, wg.s1, h.s0, h.s0), activation)
    r.results = [(m.slot, None) for m in ((h, g, u) if save else (h,))]


def gated_linear(x, w_gate, w_up, activation="silu", *, save=False):
    """act(x @ w_gate) * (x @ w_up); with save=True also the two products, for the backward pass."""
    return _call(_plan_gated_linear, (activation, bool(save)), ("x", "w_gate", "w_up"), (x, w_gate, w_up))


def _plan_gated_linear_backward(r, activation):
    _activation(activation)
    r.shape("x", tuple(r.tensors["dh"].shape[:-1]) + tuple(r.tensors["x"].shape[-1:]))
    x = r.rows("x")
    originals = r.matrix("w_gate", x.cols), r.matrix("w_up", x.cols)
    wg, wu = _gated_weights(r, x.cols)
    r.shape("dh", tuple(r.tensors["x"].shape[:-1]) + (wg.cols,))
    for name in ("pre_gate", "pre_up"):
        r.shape(name, r.tensors["dh"].shape)
    dh, g, u = r.rows("dh"), r.rows("pre_gate"), r.rows("pre_up")
    if g.s0 != u.s0:
        g, u = r.rows("pre_gate", dense=True), r.rows("pre_up", dense=True)
    M, N, K = x.rows, wg.cols, x.cols
    dg, du = r.new((M, N)), r.new((M, N))
    r.launch(kernels.GatedActivationBackward, dict(dout=dh, pre_gate=g, pre_up=u, dgate=dg, dup=du),
             (M, N, dh.s0, g.s0, dg.s0), activation)
    dx = r.new(r.tensors["x"].shape)
    a, b = wg.T, wu.T
    r.launch(kernels.LinearSum, dict(x=dg, w=a, x2=du, w2=b, out=dx),
             (M, K, N, dg.s0, dg.s1, a.s0, a.s1, dx.s0))
    dwg, (a, b), first = _weight_gradient(r, x, dg, originals[0])
    dwu, (a2, b2), second = _weight_gradient(r, x, du, originals[1])
    if first[1] is second[1]:
        r.launch(kernels.LinearPair, dict(x=a, w=b, x2=a2, w2=b2, out=dwg, out2=dwu),
                 (a.rows, b.cols, a.cols, a.s0, a.s1, b.s0, b.s1, dwg.s0))
    else:                               # two layouts: two products
        r.product(a, b, dwg)
        r.product(a2, b2, dwu)
    r.results = [(dx.slot, None), first, second]


def gated_linear_backward(dh, x, w_gate, w_up, pre_gate, pre_up, activation="silu"):
    """(dx, dw_gate, dw_up) of gated_linear, from the products it saved."""
    return _call(_plan_gated_linear_backward, (activation,), ("dh", "x", "w_gate", "w_up", "pre_gate", "pre_up"),
                 (dh, x, w_gate, w_up, pre_gate, pre_up))


# ---- residual norm ----------------------------------------------------------------------------------

def _norm_operands(r, D, kind):
    if kind not in ("rms", "layer"):
        raise ValueError(f"unknown norm {kind!r}; expected 'rms' or 'layer'")
    if r.tensors["weight"] is None:
        raise ValueError("the norm needs its weight")
    if r.tensors["block"] is None and (r.tensors["gate"] is not None or r.tensors["post_weight"] is not None):
        raise ValueError("a gate or a norm behind the block needs the block's output")
    return {name: r.vector(name, D) for name in ("weight", "gate", "post_weight")}


def _plan_residual_norm(r, kind, scale, eps, stats):
    residual = r.rows("residual", dense=True)
    shape, D = r.tensors["residual"].shape, residual.cols
    operands = _norm_operands(r, D, kind)
    r.shape("block", shape)
    passed = r.tensors["block"] is None and scale == 1.0     # sum is residual itself
    total = None if passed else r.new(shape)
    normed = r.new(shape)
    if stats and not D:
        raise ValueError("rows without columns have no statistics")
    rows = r.new((residual.rows, 4), torch.float32) if stats else None
    operands.update(residual=residual, block=r.rows("block", dense=True), bias=r.vector("bias", D), sum=total,
                    normed=normed, stats=rows)
    r.launch(kernels.ResidualNorm, operands,
             (residual.rows, D, _core.float_bits(scale), _core.float_bits(eps), max(D, 1)), None, kind)
    r.results = [None if passed else (total.slot, None), (normed.slot, None)] + ([(rows.slot, None)] if stats else [])


def residual_norm(residual, block=None, weight=None, bias=None, gate=None, post_weight=None, *, kind="rms", scale=1.0,
                  eps=1e-6, stats=False):
    """(sum, normed), or (sum, normed, stats) with stats=True:

        t = norm(block) * post_weight, or block;  sum = scale * residual + gate * t
        normed = norm(sum) * weight + bias

    Without a block (and with scale 1) sum is residual itself.  stats, [rows, 4] float32, is what the
    backward pass reads: mean and 1/deviation of each row of sum, then of block."""
    out = _call(_plan_residual_norm, (kind, float(scale), float(eps), bool(stats)),
                ("residual", "block", "weight", "bias", "gate", "post_weight"),
                (residual, block, weight, bias, gate, post_weight))
    return out if out[0] is not None else (residual,) + out[1:]


def _plan_residual_norm_backward(r, kind, scale, bias):
    dn = r.rows("dnormed", dense=True)
    shape, D = r.tensors["dnormed"].shape, dn.cols
    operands = _norm_operands(r, D, kind)
    for name in ("dsum", "sum", "block"):
        r.shape(name, shape)
    r.shape("stats", (dn.rows, 4))
    block = r.rows("block", dense=True)
    stats = r.rows("stats", dense=True)
    dresidual, dweight = r.new(shape), r.new((D,))
    dblock = r.new(shape) if block is not None else None
    dbias = r.new((D,)) if bias else None
    dgate = r.new((D,)) if operands["gate"] is not None else None
    dpost = r.new((D,)) if operands["post_weight"] is not None else None
    operands.update(dnormed=dn, dsum=r.rows("dsum", dense=True), sum=r.rows("sum", dense=True), stats=stats, block=block,
                    dresidual=dresidual, dblock=dblock, dweight=dweight, dbias=dbias, dgate=dgate, dpost_weight=dpost)
    r.launch(kernels.ResidualNormBackward, operands, (dn.rows, D, _core.float_bits(scale), max(D, 1)), None, kind)
    r.results = [None if m is None else (m.slot, None) for m in (dresidual, dblock, dweight, dbias, dgate, dpost)]


def residual_norm_backward(dnormed, dsum, total, stats, weight, block=None, gate=None, post_weight=None, *, kind="rms",
                           scale=1.0, bias=False):
    """(dresidual, dblock, dweight, dbias, dgate, dpost_weight) of residual_norm, None where the operand
    was not there.  dsum, the gradient that reaches sum past the norm, may be None."""
    return _call(_plan_residual_norm_backward, (kind, float(scale), bool(bias)),
                 ("dnormed", "dsum", "sum", "stats", "weight", "block", "gate", "post_weight"),
                 (dnormed, dsum, total, stats, weight, block, gate, post_weight))
