"""The feed-forward operators against their definitions in 64 bits.

Tolerances, element by element, for T with half a step h = finfo(T).eps / 2 (relative):
  * one rounding of the result: h |result| (half the smallest subnormal where f16 underflows);
  * a sum of n products in fp32, in any order, a step of which may be truncated: n 2^-23 sum |a b|;
  * an activation's slope is at most 1.13 (gelu), so an error of its argument grows by that much; its
    own evaluation errs by a few units of fp32 in the argument's magnitude: 2^-18 (1 + |z|) where fast
    exponentials are used (16-bit types), 2^-21 (1 + |z|) for f32;
  * a 16-bit gradient of a pre-activation is rounded before the products that read it: h |dz| |w|.
"""

import math

import pytest

torch = pytest.importorskip("torch")

from tmtest import require_gpu  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
SLOPE = 1.13


@pytest.fixture(scope="module")
def F():
    require_gpu()
    from triton_metal import functional
    yield functional
    functional.release()


def half(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, name):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "sigmoid": lambda: torch.sigmoid(z), "gelu": lambda: z * torch.special.ndtr(z),
            "gelu_tanh": lambda: z / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))}[name]()


def own_error(z, dtype):
    return (2.0 ** (-21 if dtype == torch.float32 else -18)) * (1 + z.abs())


def check(got, want, slack, what=""):
    """|got - want| <= one rounding of want (moved by the slack) + slack, everywhere."""
    assert got.shape == want.shape, what
    dtype = got.dtype
    h, tiny = half(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    limit = h * (want.abs() + slack) + slack + tiny
    error = (got.double() - want).abs()
    over = error > limit
    over |= ~torch.isfinite(got.double())
    if over.any():
        at = tuple(int(i) for i in over.nonzero()[0])
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} off, first at {at}: got {float(got[at])}, "
                             f"want {float(want[at])}, error {float(error[at])}, allowed {float(limit[at])}")


def normal(*shape, dtype, std=1.0, mean=0.0, seed=[0]):
    seed[0] += 1
    g = torch.Generator(device="cuda")
    g.manual_seed(seed[0])
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, std, generator=g).to(dtype)


def weight(K, N, dtype, layout):
    if layout == "nk":
        return normal(N, K, dtype=dtype, std=max(K, 1) ** -0.5).t()
    w = normal(K, N + (8 if layout == "padded" else 0), dtype=dtype, std=max(K, 1) ** -0.5)
    return w[:, :N]


# M, K, N: one element, single rows and columns, tile edges of every kernel (16, 64, 128, 256), odd
# sizes, sizes that reach the narrow, the wide and the unaligned paths
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 4096, 1024), (3, 17, 5), (16, 256, 640), (17, 72, 136), (33, 1000, 264),
          (64, 64, 2048), (128, 2056, 128), (129, 136, 1000), (200, 65, 129), (256, 512, 256), (257, 1024, 520),
          (513, 320, 1032), (1000, 88, 776), (300, 2049, 515), (1024, 4096, 2048), (1, 0, 9), (5, 8, 1), (1, 1031, 4099)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["kn", "nk", "padded"])
def test_linear(F, shape, element, layout):
    M, K, N = shape
    dtype = TYPES[element]
    # the activation and the operands vary with the case
    pick = (M + 3 * K + 5 * N + len(layout) + len(element))
    name = ACTIVATIONS[pick % 6]
    x = normal(M, K + 8, dtype=dtype)[:, :K] if pick % 2 else normal(M, K, dtype=dtype)
    w = weight(K, N, dtype, layout)
    bias = normal(N, dtype=dtype, std=0.3) if pick % 3 else None
    residual = normal(M, N + 3, dtype=dtype)[:, :N] if pick % 4 == 1 else (normal(M, N, dtype=dtype) if pick % 4 else None)
    out, pre = F.linear(x, w, bias, residual, activation=name, pre=True)
    z = x.double() @ w.double()
    slack = (K + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs())
    if bias is not None:
        z = z + bias.double()
        slack = slack + 2.0 ** -23 * (z.abs() + bias.double().abs())
    check(pre, z, slack, "pre")
    want = act64(z, name)
    slack = SLOPE * slack + own_error(z, dtype)
    if residual is not None:
        want = want + residual.double()
        slack = slack + 2.0 ** -23 * want.abs()
    check(out, want, slack, "out")
    again = F.linear(x, w, bias, residual, activation=name)
    assert torch.equal(again, out)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_gated_linear(F, shape, element, layout):
    M, K, N = shape
    dtype = TYPES[element]
    name = ACTIVATIONS[(M + 3 * K + 5 * N + len(layout) + len(element)) % 6]
    x, wg, wu = normal(M, K, dtype=dtype), weight(K, N, dtype, layout), weight(K, N, dtype, layout)
    h, g, u = F.gated_linear(x, wg, wu, activation=name, save=True)
    eg = (K + 2) * 2.0 ** -23 * (x.double().abs() @ wg.double().abs())
    eu = (K + 2) * 2.0 ** -23 * (x.double().abs() @ wu.double().abs())
    g64, u64 = x.double() @ wg.double(), x.double() @ wu.double()
    check(g, g64, eg, "gate")
    check(u, u64, eu, "up")
    a, ea = act64(g64, name), SLOPE * eg + own_error(g64, dtype)
    check(h, a * u64, ea * (u64.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u64).abs(), "h")
    assert torch.equal(F.gated_linear(x, wg, wu, activation=name), h)


def dact64(z, name):
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(act64(z, name).sum(), z)[0]


def product_slack(a, ea, b, K):
    """Error of a @ b where a errs by ea: the operands' and the sum's."""
    return ea @ b.abs() + (K + 2) * 2.0 ** -23 * ((a.abs() + ea) @ b.abs())


BACKWARD = [(1, 64, 64), (3, 17, 5), (16, 256, 640), (77, 520, 264), (128, 128, 256), (129, 136, 1000), (513, 320, 1032),
            (1000, 88, 776), (300, 1025, 515), (2048, 512, 1024), (1, 1, 1), (0, 16, 24), (5, 8, 1)]


@pytest.mark.parametrize("shape", BACKWARD, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_linear_backward(F, shape, element, layout):
    M, K, N = shape
    dtype = TYPES[element]
    name = ACTIVATIONS[(M + 3 * K + 5 * N + len(layout) + len(element)) % 6]
    x, w, dout = normal(M, K, dtype=dtype), weight(K, N, dtype, layout), normal(M, N, dtype=dtype)
    pre = normal(M, N, dtype=dtype)
    dx, dw, db = F.linear_backward(dout, x, w, pre, activation=name, bias=True)
    assert _by_rows(dw) == _by_rows(w) or 1 in dw.shape
    d = dact64(pre.double(), name)
    dz = dout.double() * d
    own = dout.double().abs() * own_error(pre.double(), dtype) if name != "none" else torch.zeros_like(dz)
    check(db, dz.sum(0), own.sum(0) + (M + 8) * 2.0 ** -23 * dz.abs().sum(0), "db")
    stored = own + (half(dtype) * (dz.abs() + own) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
                    if name != "none" else 0)
    check(dx, dz @ w.double().t(), product_slack(dz, stored, w.double().t(), N), "dx")
    check(dw, x.double().t() @ dz, product_slack(dz.t(), stored.t(), x.double(), M).t(), "dw")


def _by_rows(w):
    return w.stride(1) == 1


@pytest.mark.parametrize("shape", BACKWARD, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_gated_linear_backward(F, shape, element, layout):
    M, K, N = shape
    dtype = TYPES[element]
    name = ACTIVATIONS[(M + 3 * K + 5 * N + len(layout) + len(element)) % 6]
    x, wg, wu = normal(M, K, dtype=dtype), weight(K, N, dtype, layout), weight(K, N, dtype, layout)
    dh, g, u = (normal(M, N, dtype=dtype) for _ in range(3))
    dx, dwg, dwu = F.gated_linear_backward(dh, x, wg, wu, g, u, activation=name)
    g64, u64, dh64 = g.double(), u.double(), dh.double()
    dg, du = dh64 * u64 * dact64(g64, name), dh64 * act64(g64, name)
    h, tiny = half(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    own = own_error(g64, dtype)
    eg = (dh64 * u64).abs() * own + h * dg.abs() * 1.01 + 2.0 ** -22 * dg.abs() + tiny
    eu = dh64.abs() * own + h * du.abs() * 1.01 + 2.0 ** -22 * du.abs() + tiny
    a, b = wg.double().t(), wu.double().t()
    both = product_slack(dg, eg, a, N) + product_slack(du, eu, b, N)
    both = both + (N + 2) * 2.0 ** -23 * (dg.abs() @ a.abs() + du.abs() @ b.abs())      # one sum of 2N products
    check(dx, dg @ a + du @ b, both, "dx")
    check(dwg, x.double().t() @ dg, product_slack(dg.t(), eg.t(), x.double(), M).t(), "dwg")
    check(dwu, x.double().t() @ du, product_slack(du.t(), eu.t(), x.double(), M).t(), "dwu")


# ---- norms -----------------------------------------------------------------------------------------

EPS = 1e-6
DEPTH = 64      # the longest chain of fp32 additions in a row sum: 32 of a thread, 5 + 16 across threads, a few more


def norm64(v, kind):
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    return c / torch.sqrt(c.pow(2).mean(-1, keepdim=True) + EPS)


def norm_slack(v, ev, kind, n):
    """Error of norm(v) where v errs by ev: the row sums' relative error, the mean's, and v's own."""
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / torch.sqrt(c.pow(2).mean(-1, keepdim=True) + EPS)
    em = (DEPTH * 2.0 ** -24 * v.abs().mean(-1, keepdim=True) + ev.mean(-1, keepdim=True)) if kind == "layer" else 0
    e = ev + em + 2.0 ** -23 * v.abs()
    spread = (c.abs() * e).mean(-1, keepdim=True) * r * r * 1.01      # relative error of r through the row's errors
    return r * e + (c * r).abs() * (spread + DEPTH * 2.0 ** -23)


NORM_SHAPES = [(1, 4096), (5, 1), (3, 7), (4, 16), (300, 64), (129, 127), (77, 256), (65, 512), (33, 1000), (40, 1023),
               (19, 1024), (700, 2048), (9, 2050), (11, 4104), (6, 5000), (3, 8192), (2, 8191), (3, 16384), (2, 16383),
               (1300, 320)]


def norm_inputs(M, D, dtype, pick):
    block = normal(M, D, dtype=dtype, std=1.5, mean=0.2) if pick % 5 else None
    gate = normal(D, dtype=dtype, std=0.2, mean=0.5) if block is not None and pick % 2 else None
    post = normal(D, dtype=dtype, std=0.1, mean=1.0) if block is not None and pick % 3 else None
    bias = normal(D, dtype=dtype, std=0.1) if pick % 4 else None
    return block, gate, post, bias, normal(D, dtype=dtype, std=0.1, mean=1.0)


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm(F, shape, element, kind):
    M, D = shape
    dtype = TYPES[element]
    pick = M + D + len(kind) + len(element)
    block, gate, post, bias, w = norm_inputs(M, D, dtype, pick)
    r = normal(M, D, dtype=dtype, std=2.0)
    scale = 0.75 if pick % 3 == 1 else 1.0
    total, normed, stats = F.residual_norm(r, block, w, bias, gate, post, kind=kind, scale=scale, eps=EPS, stats=True)
    t, et = torch.zeros_like(r, dtype=torch.float64), torch.zeros_like(r, dtype=torch.float64)
    if block is not None:
        t = block.double()
        if post is not None:
            et = norm_slack(t, et, kind, D) * post.double().abs()
            t = norm64(t, kind) * post.double()
        if gate is not None:
            t, et = t * gate.double(), et * gate.double().abs()
    s = scale * r.double() + t
    es = et + 2.0 ** -22 * (r.double().abs() + t.abs())
    if block is None and scale == 1.0:
        assert total is r
    else:
        check(total, s, es, "sum")
    n = norm64(s, kind) * w.double()
    en = norm_slack(s, es, kind, D) * w.double().abs() + 2.0 ** -22 * n.abs()
    if bias is not None:
        n = n + bias.double()
        en = en + 2.0 ** -23 * (n.abs() + bias.double().abs())
    check(normed, n, en, "normed")
    mean = s.mean(-1) if kind == "layer" else torch.zeros(M, dtype=torch.float64, device="cuda")
    check(stats[:, 0], mean, DEPTH * 2.0 ** -24 * s.abs().mean(-1) + es.mean(-1), "mean")
    again = F.residual_norm(r, block, w, bias, gate, post, kind=kind, scale=scale, eps=EPS)
    assert torch.equal(again[1], normed)


@pytest.mark.parametrize("shape", NORM_SHAPES + [(0, 48)], ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_backward(F, shape, element, kind):
    M, D = shape
    dtype = TYPES[element]
    pick = M + 2 * D + len(kind) + len(element)
    block, gate, post, bias, w = norm_inputs(M, D, dtype, pick)
    scale = 0.75 if pick % 3 == 1 else 1.0
    s, dn = normal(M, D, dtype=dtype, std=2.0), normal(M, D, dtype=dtype)
    ds = normal(M, D, dtype=dtype) if pick % 7 else None

    def row_stats(v):
        v = v.double()
        m = v.mean(-1) if kind == "layer" else torch.zeros(M, dtype=torch.float64, device="cuda")
        return m, 1 / torch.sqrt((v - m[:, None]).pow(2).mean(-1) + EPS)

    columns = row_stats(s) + (row_stats(block) if block is not None else (torch.zeros(M, device="cuda"),) * 2)
    stats = torch.stack([c.float() for c in columns], dim=1)
    got = F.residual_norm_backward(dn, ds, s, stats, w, block, gate, post, kind=kind, scale=scale, bias=bias is not None)

    leaf = {k: v.double().requires_grad_(True) for k, v in
            dict(s=s, w=w, b=bias, y=block, g=gate, p=post).items() if v is not None}
    n = norm64(leaf["s"], kind) * leaf["w"] + (leaf["b"] if bias is not None else 0)
    first = torch.autograd.grad(n, [leaf["s"], leaf["w"]] + ([leaf["b"]] if bias is not None else []), dn.double())
    g = first[0] + (ds.double() if ds is not None else 0)
    want = [scale * g, None, first[1], first[2] if bias is not None else None, None, None]
    if block is not None:
        t = norm64(leaf["y"], kind) * leaf["p"] if post is not None else leaf["y"]
        t = t * leaf["g"] if gate is not None else t * 1.0
        names = ["y"] + (["g"] if gate is not None else []) + (["p"] if post is not None else [])
        second = dict(zip(names, torch.autograd.grad(t, [leaf[k] for k in names], g)))
        want[1], want[4], want[5] = second["y"], second.get("g"), second.get("p")
    # Every gradient is a sum of a few products of the terms below; each is formed from fp32 values whose
    # relative error is at most E (the row sums' depth, the statistics' rounding, a few operations).
    E = (2 * DEPTH + 16) * 2.0 ** -23
    if M and D:
        hat = norm64(s.double(), kind).abs() + 1e-3
        hw = dn.double().abs() * w.double().abs()
        r = torch.as_tensor(columns[1])[:, None]
        lead = r * s.double().abs().mean(-1, keepdim=True)       # what is lost in s - mean
        size = (ds.double().abs() if ds is not None else 0) + r * (hw + hw.mean(-1, keepdim=True)
                                                                    + (hat + lead) * (hw * (hat + lead)).mean(-1, keepdim=True))
        hy = dt = gy = None
        slack = [E * size, None, E * (dn.double().abs() * (hat + lead)).sum(0), E * dn.double().abs().sum(0), None, None]
        if block is not None:
            gy = gate.double().abs() if gate is not None else 1.0
            dt = size * gy
            if post is not None:
                ry = torch.as_tensor(columns[3])[:, None]
                yh = norm64(block.double(), kind).abs() + 1e-3 + ry * block.double().abs().mean(-1, keepdim=True)
                hy = dt * post.double().abs()
                slack[1] = 2 * E * ry * (hy + hy.mean(-1, keepdim=True) + yh * (hy * yh).mean(-1, keepdim=True))
                slack[4] = 2 * E * (size * yh * post.double().abs()).sum(0)
                slack[5] = 2 * E * (dt * yh).sum(0)
            else:
                slack[1] = 2 * E * dt
                slack[4] = 2 * E * (size * block.double().abs()).sum(0)
        for i in (2, 3, 4, 5):      # the sums over the rows themselves
            if slack[i] is not None:
                slack[i] = slack[i] * (1 + (M + 16) * 2.0 ** -23 / E)
    else:
        slack = [torch.zeros_like(v) if v is not None else None for v in want]
    for i, what in enumerate(("dresidual", "dblock", "dweight", "dbias", "dgate", "dpost")):
        assert (got[i] is None) == (want[i] is None), what
        if want[i] is not None:
            check(got[i], want[i], slack[i], what)


# ---- gradients against differences ---------------------------------------------------------------------

def along(f, point, direction, h):
    return (f(point + h * direction) - f(point - h * direction)) / (2 * h)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu", "sigmoid"])
def test_gradients_against_differences(F, name):
    """f32, directional: the difference errs by h^2/6 of the third derivative and by rounding / h.  With
    h = 2^-6 and outputs of size 1, rounded to 2^-24 and summed with weights of size 1 over 48 x 40
    of them, both stay under 1e-3 of the gradient's norm (about sqrt(48 x 40) here)."""
    M, K, N = 48, 56, 40
    f32 = torch.float32
    x, wg, wu, c = normal(M, K, dtype=f32), weight(K, N, f32, "kn"), weight(K, N, f32, "kn"), normal(M, N, dtype=f32)
    h, g, u = F.gated_linear(x, wg, wu, activation=name, save=True)
    grads = F.gated_linear_backward(c, x, wg, wu, g, u, activation=name)
    operands = [x, wg, wu]
    for i in range(3):
        v = normal(*operands[i].shape, dtype=f32, std=operands[i].shape[0] ** -0.5 if i else K ** -0.5)

        def loss(p):
            args = list(operands)
            args[i] = p
            return float((F.gated_linear(*args, activation=name).double() * c.double()).sum())

        want = float((grads[i].double() * v.double()).sum())
        assert abs(along(loss, operands[i], v, 2.0 ** -6) - want) < 2e-3 * math.sqrt(M * N)
    b = normal(N, dtype=f32)
    out, pre = F.linear(x, wg, b, activation=name, pre=True)
    dx, dw, db = F.linear_backward(c, x, wg, pre, activation=name, bias=True)
    for grad, p, f in ((dx, x, lambda p: F.linear(p, wg, b, activation=name)), (dw, wg, lambda p: F.linear(x, p, b, activation=name)),
                       (db, b, lambda p: F.linear(x, wg, p, activation=name))):
        v = normal(*p.shape, dtype=f32, std=0.15)
        want = float((grad.double() * v.double()).sum())
        got = along(lambda q: float((f(q).double() * c.double()).sum()), p, v, 2.0 ** -6)
        assert abs(got - want) < 2e-3 * math.sqrt(M * N)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_gradients_against_differences(F, kind):
    M, D = 24, 72
    f32 = torch.float32
    r, y = normal(M, D, dtype=f32, std=2.0), normal(M, D, dtype=f32)
    w, b, g, p = (normal(D, dtype=f32, std=0.3, mean=1.0) for _ in range(4))
    cs, cn = normal(M, D, dtype=f32), normal(M, D, dtype=f32)
    args = [r, y, w, b, g, p]
    total, normed, stats = F.residual_norm(*args, kind=kind, scale=0.5, stats=True)
    grads = F.residual_norm_backward(cn, cs, total, stats, w, y, g, p, kind=kind, scale=0.5, bias=True)
    for i, grad in enumerate(grads):
        v = normal(*args[i].shape, dtype=f32, std=0.2)

        def loss(q):
            a = list(args)
            a[i] = q
            s, n = F.residual_norm(*a, kind=kind, scale=0.5)
            return float((s.double() * cs.double() + n.double() * cn.double()).sum())

        want = float((grad.double() * v.double()).sum())
        assert abs(along(loss, args[i], v, 2.0 ** -6) - want) < 2e-3 * math.sqrt(M * D)


# ---- a run of them, as a layer uses them ------------------------------------------------------------------

def layer(F, t, dtype):
    s1, n1, st1 = F.residual_norm(t["r"], t["y"], t["w"], None, t["g"], t["p"], scale=0.5, stats=True)
    h, gate, up = F.gated_linear(n1, t["wg"], t["wu"], save=True)
    out = F.linear(h, t["wd"], None, s1)
    return out, (s1, n1, st1, h, gate, up)


def layer_backward(F, t, kept, dout):
    s1, n1, st1, h, gate, up = kept
    dh, dwd, _ = F.linear_backward(dout, h, t["wd"])
    dn, dwg, dwu = F.gated_linear_backward(dh, n1, t["wg"], t["wu"], gate, up)
    dr, dy, dw, _, dg, dp = F.residual_norm_backward(dn, dout, s1, st1, t["w"], t["y"], t["g"], t["p"], scale=0.5)
    return dict(r=dr, y=dy, w=dw, g=dg, p=dp, wg=dwg, wu=dwu, wd=dwd)


def layer_inputs(dtype, lead=(3, 70), D=256, H=704):
    t = dict(r=normal(*lead, D, dtype=dtype), y=normal(*lead, D, dtype=dtype))
    for name in ("w", "g", "p"):
        t[name] = normal(D, dtype=dtype, std=0.1, mean=1.0)
    t["wg"], t["wu"], t["wd"] = weight(D, H, dtype, "kn"), weight(D, H, dtype, "nk"), weight(H, D, dtype, "nk")
    t["wu"] = t["wu"].contiguous()
    return t


def layer64(t):
    s = 0.5 * t["r"] + t["g"] * norm64(t["y"], "rms") * t["p"]
    n = norm64(s, "rms") * t["w"]
    return s + (act64(n @ t["wg"], "silu") * (n @ t["wu"])) @ t["wd"]


@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
def test_a_layer_forward_and_backward(F, element):
    """At most ten roundings lie between the inputs and any result, each a relative 2-norm error of at
    most h; every map in between has a norm of a few, so 40 h bounds the sum of what reaches a result.
    f32 sums add 1e-6 or so of their own."""
    dtype = TYPES[element]
    t = layer_inputs(dtype)
    out, kept = layer(F, t, dtype)
    dout = normal(*out.shape, dtype=dtype)
    grads = layer_backward(F, t, kept, dout)
    leaves = {k: v.double().requires_grad_(True) for k, v in t.items()}
    want = layer64(leaves)
    wanted = dict(zip(leaves, torch.autograd.grad(want, list(leaves.values()), dout.double())))
    want = want.detach()
    limit = 40 * half(dtype) + 2e-6
    assert float((out.double() - want).norm() / want.norm()) < limit
    for k in t:
        assert grads[k].shape == t[k].shape
        assert float((grads[k].double() - wanted[k]).norm() / wanted[k].norm()) < limit, k


@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_captured_and_replayed(F, element):
    """Forward and backward in one graph; replays with other inputs give what eager calls give, also
    while another graph's replay and eager work share the device."""
    dtype = TYPES[element]
    t = layer_inputs(dtype, lead=(130,))
    dout = normal(130, 256, dtype=dtype)
    graphs, results = [], []
    side = torch.cuda.Stream()
    layer(F, t, dtype)
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, kept = layer(F, t, dtype)
            results.append((out, layer_backward(F, t, kept, dout)))
        graphs.append(graph)
    for step in range(3):
        for k in t:
            t[k].copy_(normal(*t[k].shape, dtype=dtype) if step else t[k])
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        out, kept = layer(F, t, dtype)
        grads = layer_backward(F, t, kept, dout)
        torch.cuda.synchronize()
        for got, got_grads in results:
            assert torch.equal(got, out)
            for k in grads:
                assert torch.equal(got_grads[k], grads[k]), k
    for graph in graphs:
        graph.reset()


FIRST_USE = """
import sys, torch
sys.path.insert(0, {package!r})
from triton_metal import functional as F
torch.manual_seed(0)
make = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)
x, w, r, g = make(130, 264), make(264, 200), make(130, 200), make(130, 200)
xo, wn, rn = make(130, 257), make(512), make(70, 512)
torch.cuda.synchronize()
def work():
    a = F.linear(x, w, None, r, activation="gelu")
    b = F.linear_backward(g, x, w, r, activation="silu", bias=True)
    c = F.linear(xo, make_odd)
    s, n, st = F.residual_norm(rn, rn, wn, stats=True)
    d = F.residual_norm_backward(n, None, s, st, wn, rn)
    return [a, *b, c, s, n, d[0], d[2]]
make_odd = make(257, 333)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = work()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(captured, work()))
graph.reset()
F.release()
"""


def test_the_first_use_may_be_captured(F):
    """In a process of its own: nothing has been loaded, probed or sized before the capture begins."""
    import pathlib
    import subprocess
    import sys
    package = str(pathlib.Path(__file__).resolve().parents[1] / "triton-metal_b200")
    done = subprocess.run([sys.executable, "-c", FIRST_USE.format(package=package)], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_streams_at_once(F):
    dtype = torch.bfloat16
    sets = [(normal(2048, 512, dtype=dtype), weight(512, 1024, dtype, "kn"), normal(2048, 1024, dtype=dtype),
             normal(2048, 1024, dtype=dtype)) for _ in range(2)]
    want = [F.linear_backward(d, x, w, z, activation="gelu", bias=True) for x, w, d, z in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (x, w, d, z) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(F.linear_backward(d, x, w, z, activation="gelu", bias=True))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))


# ---- memory that is not the operators' -----------------------------------------------------------------

@pytest.mark.parametrize("element", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(3, 64, 40), (130, 264, 136), (300, 128, 72), (200, 65, 33), (257, 1024, 520)], ids=str)
def test_padding_columns_and_rows_stay(F, element, shape):
    M, K, N = shape
    dtype = TYPES[element]
    x, w = normal(M, K, dtype=dtype), weight(K, N, dtype, "kn")
    wide = torch.full((M + 2, N + 16), 7.0, dtype=dtype, device="cuda")
    F.linear(x, w, out=wide[:M, :N])
    assert torch.equal(wide[:M, :N], F.linear(x, w))
    assert (wide[M:] == 7).all() and (wide[:, N:] == 7).all()


@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_broadcast_operands(F, element):
    """Strides of zero: one row of x, of the residual or of a gradient for all rows, one column of w for all columns."""
    dtype = TYPES[element]
    for M, K, N in ((5, 64, 72), (300, 256, 264), (140, 65, 33)):
        x, r = normal(1, K, dtype=dtype).expand(M, K), normal(N, dtype=dtype).expand(M, N)
        w, flat = weight(K, N, dtype, "kn"), normal(K, 1, dtype=dtype).expand(K, N)
        assert torch.equal(F.linear(x, w, None, r), F.linear(x.contiguous(), w, None, r.contiguous()))
        y = normal(M, K, dtype=dtype)
        slack = (K + 2) * 2.0 ** -23 * (y.double().abs() @ flat.double().abs())
        check(F.linear(y, flat), y.double() @ flat.double(), slack)
        for got, want in zip(F.linear_backward(r, y, w), F.linear_backward(r.contiguous(), y, w)):
            assert got is want is None or torch.equal(got, want)
        wn = normal(K, dtype=dtype)
        for got, want in zip(F.residual_norm(x, y, wn), F.residual_norm(x.contiguous(), y, wn)):
            assert torch.equal(got, want)


def test_more_than_two_dimensions_and_views(F):
    dtype = torch.bfloat16
    base = normal(4, 6, 2, 128, dtype=dtype)
    w = weight(128, 136, dtype, "nk")
    for x in (base, base.transpose(0, 1), base[:, ::2], base[..., ::2, :], base[0, 0, 0]):
        got = F.linear(x, w)
        assert got.shape == x.shape[:-1] + (136,)
        assert torch.equal(got.reshape(-1, 136), F.linear(x.reshape(-1, 128).contiguous(), w))
        dx, dw, _ = F.linear_backward(got, x, w)
        assert dx.shape == x.shape and dw.shape == w.shape
    columns = normal(64, 300, dtype=dtype)[:, ::2]                   # no unit stride
    assert torch.equal(F.linear(columns[:, :128], w), F.linear(columns[:, :128].contiguous(), w))
    no_unit = normal(256, 272, dtype=dtype)[::2, ::2]
    assert torch.equal(F.linear(base, no_unit), F.linear(base, no_unit.contiguous()))
    mixed = F.gated_linear(base, w, w.contiguous())                  # two layouts in one call
    assert torch.equal(mixed, F.gated_linear(base, w.contiguous(), w.contiguous()))


def test_side_by_side_outputs(F):
    """Two results as the column halves of one tensor, through the C entry: rows interleave, nothing overlaps."""
    from triton_metal import kernels
    M, K, N = 200, 128, 96
    dtype = torch.bfloat16
    x, wg, wu = normal(M, K, dtype=dtype), weight(K, N, dtype, "kn"), weight(K, N, dtype, "kn")
    both, h = torch.zeros(M, 2 * N, dtype=dtype, device="cuda"), torch.zeros(M, N, dtype=dtype, device="cuda")
    kern = kernels.GatedLinear("bf16", ("pre_gate", "pre_up"), "silu")
    try:
        tensors = [x, wg, wu, h, both[:, :N], both[:, N:]]
        size = [t.untyped_storage().nbytes() - t.storage_offset() * 2 for t in tensors]
        kern.launch_tensors(torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in tensors], size,
                            (M, N, K, K, 1, N, 1, N, 2 * N))
        want = F.gated_linear(x, wg, wu, save=True)
        assert torch.equal(h, want[0]) and torch.equal(both[:, :N], want[1]) and torch.equal(both[:, N:], want[2])
    finally:
        kern.release()


def test_in_place_norms(F):
    from triton_metal import _core, kernels
    for M, D in ((7, 96), (300, 1024), (500, 4096), (40, 1023)):
        dtype = torch.bfloat16
        r, y, w = normal(M, D, dtype=dtype), normal(M, D, dtype=dtype), normal(D, dtype=dtype)
        want = F.residual_norm(r, y, w, scale=0.5)
        kern = kernels.ResidualNorm("bf16", ("block", "sum"))
        try:
            # REQUIRED (residual, weight, normed), then block, sum: the sum over the residual, the norm over the block
            tensors = [r, w, y, y, r]
            kern.launch_tensors(torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in tensors],
                                [t.nbytes for t in tensors], (M, D, _core.float_bits(0.5), _core.float_bits(1e-6), D))
            assert torch.equal(r, want[0]) and torch.equal(y, want[1])
        finally:
            kern.release()


def test_in_place_residual(F):
    for M, K, N in ((5, 64, 72), (300, 256, 264), (130, 65, 33)):
        x, w, r = normal(M, K, dtype=torch.bfloat16), weight(K, N, torch.bfloat16, "kn"), normal(M, N, dtype=torch.bfloat16)
        want = F.linear(x, w, None, r, activation="silu")
        got = F.linear(x, w, None, r, activation="silu", out=r)
        assert got is r and torch.equal(r, want)


@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_a_nan_or_infinity_stays_in_its_row(F, element):
    dtype = TYPES[element]
    for M, K, N in ((7, 64, 72), (200, 256, 264), (140, 65, 33)):
        x, w = normal(M, K, dtype=dtype), weight(K, N, dtype, "kn")
        clean = F.linear(x, w, activation="relu")
        x[3, 5] = float("nan")
        x[4, 6] = float("inf")
        out = F.linear(x, w, activation="relu")
        assert out[3].isnan().all()
        assert torch.equal(out[5:], clean[5:]) and torch.equal(out[:3], clean[:3])
        assert (torch.isinf(out[4]) | (out[4] == 0)).all()
    r, wn = normal(9, 264, dtype=dtype), normal(264, dtype=dtype)
    clean = F.residual_norm(r, None, wn)[1]
    r[2, 7] = float("nan")
    got = F.residual_norm(r, None, wn)[1]
    assert got[2].isnan().all() and torch.equal(got[3:], clean[3:])


def test_far_offsets(F):
    """Rows whose offset passes 2^31 elements: a column slice of a tensor of 2^31 + elements."""
    rows, pitch, D = 4100, 1 << 19, 256
    wide = torch.empty(rows, pitch, dtype=torch.bfloat16, device="cuda")
    x = wide[:, :D]
    x.normal_()
    w = weight(D, 264, torch.bfloat16, "kn")
    assert torch.equal(F.linear(x, w), F.linear(x.contiguous(), w))
    out = wide[:, 512:512 + 264]
    F.linear(x, w, out=out)
    assert torch.equal(out, F.linear(x.contiguous(), w))
    tail = wide[-3:, :D]
    assert torch.equal(F.linear(tail, w), F.linear(tail.contiguous(), w))


# ---- buffers and tm_launch -----------------------------------------------------------------------------

def test_buffers_grid_and_timed_launches(core, no_leaks):
    import numpy as np

    from triton_metal import cuda, kernels
    from triton_metal.buffer import MetalBuffer
    M, K, N = 200, 96, 150
    rng = np.random.default_rng(3)
    x, w, b = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N), (N,)))
    bufs = [MetalBuffer.from_numpy(a) for a in (x, w, b)] + [MetalBuffer.from_numpy(np.full((M, N), 9, np.float32))]
    kern = kernels.Linear("f32", ("bias",), "relu", block=(64, 32))
    operands = dict(zip(("x", "w", "bias", "out"), (buf.tm_handle for buf in bufs)))
    try:
        grid, kinds, values = kern.arguments(**operands, M=M, N=N, K=K)
        assert grid == (4, 5, 1)
        kern.launch((2, 3, 1), kinds, values)              # programs beyond the grid are not computed
        got = bufs[3].numpy()
        want = np.maximum(x.astype(np.float64) @ w + b, 0)
        assert np.abs(got[:128, :96] - want[:128, :96]).max() < (K + 4) * 2.0 ** -23 * 4 * K
        assert (got[128:] == 9).all() and (got[:, 96:] == 9).all()
        kern(**operands, M=M, N=N, K=K)
        assert np.abs(bufs[3].numpy() - want).max() < (K + 4) * 2.0 ** -23 * 4 * K
        before = cuda.launch_count()
        assert kern.time(grid, kinds, values, 3) > 0 and cuda.launch_count() == before + 3
        kern.launch_async(grid, kinds, values)
        cuda.synchronize()
        # a buffer handle is ordered by the library's stream and by no other
        c_kinds, c_values, n = core.pack_arguments(kinds, values)
        lengths = (type(c_values)._type_ * n)()
        import torch
        stream = torch.cuda.Stream().cuda_stream
        assert cuda._lib.tmx_launch_on(kern.handle, stream, *grid, 128, c_kinds, c_values, lengths, n) == -1
        assert "ordered by the library's stream" in core.last_error()
        assert cuda._lib.tmx_launch_on(kern.handle, cuda.stream_handle(), *grid, 128, c_kinds, c_values, lengths, n) == 0
        cuda.synchronize()
    finally:
        kern.release()
        for buf in bufs:
            buf.free()


def test_norm_and_activation_gradients_through_buffers(core, no_leaks):
    import numpy as np

    from triton_metal import kernels
    from triton_metal.buffer import MetalBuffer
    M, D = 70, 96
    rng = np.random.default_rng(4)
    made = {}

    def put(name, *shape):
        made[name] = MetalBuffer.from_numpy(rng.standard_normal(shape).astype(np.float32))
        return made[name].tm_handle

    norm = kernels.ResidualNorm("f32", ("block", "sum", "stats"), None, "layer")
    act = kernels.ActivationBackward("f32", ("pre", "dz", "dbias"), "silu", block=(32, 128))
    try:
        norm(residual=put("r", M, D), weight=put("w", D), normed=put("n", M, D), block=put("y", M, D), sum=put("s", M, D),
             stats=put("st", M, 4), scale=0.5, eps=1e-5, M=M, D=D)
        get = lambda k: made[k].numpy().astype(np.float64)  # noqa: E731
        s = 0.5 * get("r") + get("y")
        mean, var = s.mean(1, keepdims=True), s.var(1, keepdims=True)
        assert np.abs(get("s") - s).max() < 2e-6
        assert np.abs(get("n") - (s - mean) / np.sqrt(var + 1e-5) * get("w")).max() < 2e-5
        assert np.abs(get("st")[:, 0] - mean[:, 0]).max() < 1e-6
        act(dout=put("d", M, D), pre=put("z", M, D), dz=put("dz", M, D), dbias=put("db", D), M=M, N=D)
        z = get("z")
        sig = 1 / (1 + np.exp(-z))
        dz = get("d") * sig * (1 + z * (1 - sig))
        assert np.abs(get("dz") - dz).max() < 1e-5 and np.abs(get("db") - dz.sum(0)).max() < 1e-4
        # a grid of one row of blocks leaves the rows behind it
        made["dz"].copy_from(np.full((M, D), 5, np.float32).ctypes.data)
        grid, kinds, values = act.arguments(dout=made["d"].tm_handle, pre=made["z"].tm_handle, dz=made["dz"].tm_handle,
                                            dbias=made["db"].tm_handle, M=M, N=D)
        act.launch((1, 1, 1), kinds, values)
        assert (get("dz")[32:] == 5).all() and np.abs(get("db") - dz[:32].sum(0)).max() < 1e-4
    finally:
        norm.release()
        act.release()
        for buf in made.values():
            buf.free()


# ---- refusals -----------------------------------------------------------------------------------------

def test_refusals(F):
    x, w = normal(4, 16, dtype=torch.bfloat16), weight(16, 24, torch.bfloat16, "kn")
    with pytest.raises(TypeError, match="bias is torch.float32"):
        F.linear(x, w, torch.zeros(24, device="cuda"))
    with pytest.raises(ValueError, match="weight has shape"):
        F.linear(x, w.t())
    with pytest.raises(ValueError, match="residual has shape"):
        F.linear(x, w, None, normal(4, 23, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="unknown activation"):
        F.linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="is on cpu"):
        F.linear(x.cpu(), w)
    with pytest.raises(ValueError, match="w_up is on cpu"):
        F.gated_linear(x, w, w.cpu())
    with pytest.raises(TypeError, match="float64"):
        F.linear(x.double(), w)
    with pytest.raises(RuntimeError, match="out overlaps its input x"):
        F.linear(x, weight(16, 16, torch.bfloat16, "kn"), out=x)
    with pytest.raises(ValueError, match="needs the pre-activations"):
        F.linear_backward(normal(4, 24, dtype=torch.bfloat16), x, w, activation="relu")
    with pytest.raises(ValueError, match="needs the block's output"):
        F.residual_norm(x, None, w[:, 0].contiguous(), gate=w[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="at most 16384 columns"):
        F.residual_norm(normal(1, 16392, dtype=torch.bfloat16), None, normal(16392, dtype=torch.bfloat16))
    from triton_metal import kernels
    kern = kernels.Linear("f32")
    try:
        host = torch.zeros(64)
        a = torch.zeros(64, device="cuda")
        with pytest.raises(RuntimeError, match="is not memory of device"):
            kern.launch_tensors(0, [host.data_ptr(), a.data_ptr(), a.data_ptr() + 128], [256, 256, 128],
                                (4, 4, 4, 4, 1, 4, 1, 4, 4, 4))
    finally:
        kern.release()
