"""The feed-forward operators where the other tests do not reach: operands in two layouts, tiles behind the first
of a CTA pair, every tile width, values at the ends of a type's range, calls of several threads.  Against the
definitions in 64 bits; the tolerances are those of test_feed_forward_gpu.py."""

import pytest

torch = pytest.importorskip("torch")

from ffn_shapes import FEW_ROWS, PAIRS  # noqa: E402
from test_feed_forward_gpu import (F, TYPES, act64, check, dact64, half, normal, own_error, product_slack,  # noqa: E402,F401
                                   weight, SLOPE)

pytestmark = pytest.mark.gpu


def gated_backward64(dh, x, wg, wu, g, u, name):
    """(wanted, slack) of dx, dw_gate, dw_up."""
    dtype, (M, N), K = dh.dtype, dh.shape, x.shape[1]
    g64, u64, dh64 = g.double(), u.double(), dh.double()
    dg, du = dh64 * u64 * dact64(g64, name), dh64 * act64(g64, name)
    h, tiny = half(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    own = own_error(g64, dtype)
    eg = (dh64 * u64).abs() * own + h * dg.abs() * 1.01 + 2.0 ** -22 * dg.abs() + tiny
    eu = dh64.abs() * own + h * du.abs() * 1.01 + 2.0 ** -22 * du.abs() + tiny
    a, b = wg.double().t(), wu.double().t()
    both = product_slack(dg, eg, a, N) + product_slack(du, eu, b, N)
    both = both + (N + 2) * 2.0 ** -23 * (dg.abs() @ a.abs() + du.abs() @ b.abs())
    x64 = x.double()
    return ((dg @ a + du @ b, both), (x64.t() @ dg, product_slack(dg.t(), eg.t(), x64, M).t()),
            (x64.t() @ du, product_slack(du.t(), eu.t(), x64, M).t()))


@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layouts", [("kn", "nk"), ("nk", "kn")], ids=str)
def test_gated_weights_in_two_layouts(F, element, layouts):
    dtype = TYPES[element]
    for M, K, N in ((24, 40, 56), (140, 264, 136), (33, 65, 31)):
        x, dh, g, u = normal(M, K, dtype=dtype), *(normal(M, N, dtype=dtype) for _ in range(3))
        wg, wu = (weight(K, N, dtype, layout) for layout in layouts)
        got = F.gated_linear_backward(dh, x, wg, wu, g, u, activation="silu")
        for t, w, (want, slack) in zip(got, (x, wg, wu), gated_backward64(dh, x, wg, wu, g, u, "silu")):
            check(t, want, slack)
            assert t.stride() == w.stride()


# ---- every kernel and tile of the 16-bit products -----------------------------------------------------------
# (test_feed_forward_choice.py holds the shapes to what they are here for.)

def products(kind, x, w, x2, w2, out_shape):
    """LinearSum or LinearPair through the C entry, on any two strides of either operand."""
    from triton_metal import kernels
    element = {torch.bfloat16: "bf16", torch.float16: "f16"}[x.dtype]
    kern = getattr(kernels, kind)(element)
    outs = [torch.full(out_shape, 7.0, device="cuda", dtype=x.dtype) for _ in range(1 if kind == "LinearSum" else 2)]
    try:
        tensors = [x, w, x2, w2] + outs
        M, K = x.shape
        kern.launch_tensors(torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in tensors],
                            [t.numel() * t.element_size() for t in tensors],
                            (M, w.shape[1], K, *x.stride(), *w.stride(), outs[0].stride(0)))
        torch.cuda.synchronize()
    finally:
        kern.release()
    return outs


def product64(x, w):
    x, w = x.double(), w.double()
    return x @ w, (x.shape[1] + 2) * 2.0 ** -23 * (x.abs() @ w.abs())


def check_case(F, mode, M, N, K, epilogue, dtype, layout):
    if mode == "linear":
        x, w = normal(M, K, dtype=dtype), weight(K, N, dtype, layout)
        z, slack = product64(x, w)
        if not epilogue:
            return check(F.linear(x, w), z, slack)
        bias, r = normal(N, dtype=dtype, std=0.3), normal(M, N, dtype=dtype)
        out, pre = F.linear(x, w, bias, r, activation="gelu", pre=True)
        z = z + bias.double()
        slack = slack + 2.0 ** -23 * (z.abs() + bias.double().abs())
        check(pre, z, slack, "pre")
        want = act64(z, "gelu") + r.double()
        return check(out, want, SLOPE * slack + own_error(z, dtype) + 2.0 ** -23 * want.abs(), "out")
    if mode == "gated":
        x, wg, wu = normal(M, K, dtype=dtype), weight(K, N, dtype, layout), weight(K, N, dtype, layout)
        (g, eg), (u, eu) = product64(x, wg), product64(x, wu)
        got = F.gated_linear(x, wg, wu, activation="gelu" if epilogue else "silu", save=bool(epilogue))
        name = "gelu" if epilogue else "silu"
        if epilogue:
            check(got[1], g, eg, "gate")
            check(got[2], u, eu, "up")
            got = got[0]
        a, ea = act64(g, name), SLOPE * eg + own_error(g, dtype)
        return check(got, a * u, ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs(), "h")
    if mode == "sum":
        x, x2 = normal(M, K, dtype=dtype), normal(M, K, dtype=dtype)
        w, w2 = weight(K, N, dtype, layout), weight(K, N, dtype, layout)
        (a, ea), (b, eb) = product64(x, w), product64(x2, w2)
        both = (K + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs() + x2.double().abs() @ w2.double().abs())
        return check(products("LinearSum", x, w, x2, w2, (M, N))[0], a + b, ea + eb + both)
    x, x2 = normal(K, M, dtype=dtype).t(), normal(K, M, dtype=dtype).t()        # x^T dz: contiguous along m
    w, w2 = (weight(K, N, dtype, layout) for _ in range(2))
    for got, (want, slack) in zip(products("LinearPair", x, w, x2, w2, (M, N)), (product64(x, w), product64(x2, w2))):
        check(got, want, slack)


@pytest.mark.parametrize("case", PAIRS, ids=str)
@pytest.mark.parametrize("element,layout", [("bf16", "kn"), ("f16", "nk")])
def test_tiles_of_the_cta_pairs(F, case, element, layout):
    mode, M, N, K, epilogue = case[:5]
    check_case(F, mode, M, N, K, epilogue, TYPES[element], layout)


@pytest.mark.parametrize("case", FEW_ROWS, ids=str)
@pytest.mark.parametrize("element,layout", [("bf16", "nk"), ("f16", "kn")])
def test_tiles_of_the_few_row_kernel(F, case, element, layout):
    mode, M, N, K = case[:4]
    check_case(F, mode, M, N, K, "pre" if mode != "sum" and M % 2 else "", TYPES[element], layout)


# ---- several host threads ---------------------------------------------------------------------------------

def test_threads_on_their_own_streams(F):
    """First calls and later ones, each thread on its own stream and operands: the results of calls made alone, and
    every launch counted."""
    import threading

    from triton_metal import cuda
    dtype, count, rounds = torch.bfloat16, 8, 100
    sets = []
    for i in range(count):
        M, K, N = 5 + i, 64 + 8 * (i % 3), 72 + 16 * (i % 2)
        sets.append(dict(x=normal(M, K, dtype=dtype), w=weight(K, N, dtype, "kn"), r=normal(M, N, dtype=dtype),
                         n=normal(N, dtype=dtype), d=normal(M, N, dtype=dtype)))

    def work(t):
        out, pre = F.linear(t["x"], t["w"], t["n"], t["r"], activation="silu", pre=True)
        total, normed, stats = F.residual_norm(out, t["r"], t["n"], scale=0.5, stats=True)
        back = F.residual_norm_backward(t["d"], t["r"], total, stats, t["n"], t["r"], scale=0.5)
        return [out, normed, back[0], back[2], *F.linear_backward(t["d"], t["x"], t["w"], pre, activation="silu", bias=True)]

    F.release()
    torch.cuda.synchronize()
    got, failed, gate = [[] for _ in sets], [], threading.Barrier(count)
    before = cuda.launch_count()

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                for _ in range(rounds):
                    got[i] = work(sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    made = cuda.launch_count() - before
    start, alone = cuda.launch_count(), [work(t) for t in sets]
    assert made == rounds * (cuda.launch_count() - start)
    for a, b in zip(got, alone):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- what earlier work leaves behind ------------------------------------------------------------------------

LEFTOVERS = [(1, 64, 64), (3, 17, 5), (16, 256, 640), (77, 520, 264), (129, 136, 1000), (300, 1025, 515), (513, 320, 1032),
             (40, 1023, 65)]


@pytest.mark.parametrize("shape", LEFTOVERS, ids=str)
@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
def test_leftovers_in_memory_do_not_reach_a_result(F, element, shape):
    """The same call before and after one on NaN throughout, which leaves NaN in the scratch memory, the temporaries,
    the outputs' memory, shared memory and TMEM that the next call is given."""
    M, K, N = shape
    dtype = TYPES[element]

    def call(t):
        out = [F.linear(t["x"], t["w"], t["b"], t["d"], activation="gelu"), *F.linear_backward(t["d"], t["x"], t["w"], t["z"],
                                                                                             activation="silu", bias=True),
               *F.gated_linear(t["x"], t["w"], t["v"], save=True),
               *F.gated_linear_backward(t["d"], t["x"], t["w"], t["v"], t["z"], t["u"])]
        total, normed, stats = F.residual_norm(t["x"], t["y"], t["n"], kind="layer", post_weight=t["n"], stats=True)
        back = F.residual_norm_backward(t["y"], t["x"], total, stats, t["n"], t["y"], post_weight=t["n"], kind="layer", bias=True)
        return [v for v in out + [total, normed, stats, *back] if v is not None]

    t = dict(x=normal(M, K, dtype=dtype), y=normal(M, K, dtype=dtype), n=normal(K, dtype=dtype), b=normal(N, dtype=dtype),
             w=weight(K, N, dtype, "kn"), v=weight(K, N, dtype, "nk"),
             **{k: normal(M, N, dtype=dtype) for k in "dzu"})
    first = [v.clone() for v in call(t)]
    assert all(torch.isfinite(v).all() for v in first)
    for _ in range(3):
        call({k: torch.full_like(v, float("nan")) for k, v in t.items()})
        assert all(torch.equal(a, b) for a, b in zip(first, call(t)))


# ---- in place ----------------------------------------------------------------------------------------------

def launch(cls, operands, scalars, element, activation=None, norm=None):
    """A kernel class on torch tensors by operand name (None is left out), on the current stream."""
    present = {k: v for k, v in operands.items() if v is not None}
    kern = cls(element, tuple(n for n in cls.OPTIONAL if n in present), activation, norm)
    try:
        tensors = [present[n] for n in kern.pointers]
        kern.launch_tensors(torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in tensors],
                            [t.numel() * t.element_size() for t in tensors], scalars)
        torch.cuda.synchronize()
    finally:
        kern.release()


IN_PLACE = [(1, 8), (7, 96), (70, 33), (300, 1024), (130, 4104), (40, 1023)]


@pytest.mark.parametrize("element", ["bf16", "f32"])
@pytest.mark.parametrize("shape", IN_PLACE, ids=str)
def test_in_place_activation_gradients(F, element, shape):
    from triton_metal import kernels
    M, N = shape
    dtype = TYPES[element]
    d, z, u = (normal(M, N, dtype=dtype) for _ in range(3))
    scalars = (M, N, N, N, N)
    want, sums = torch.empty_like(d), torch.empty_like(d[0])
    launch(kernels.ActivationBackward, dict(dout=d, pre=z, dz=want, dbias=sums), scalars, element, "gelu")
    for which in (0, 1):
        t, got = [d.clone(), z.clone()], torch.empty_like(sums)
        launch(kernels.ActivationBackward, dict(dout=t[0], pre=t[1], dz=t[which], dbias=got), scalars, element, "gelu")
        assert torch.equal(t[which], want) and torch.equal(got, sums)
        assert torch.equal(t[1 - which], (z, d)[which])
    dg, du = torch.empty_like(d), torch.empty_like(d)
    launch(kernels.GatedActivationBackward, dict(dout=d, pre_gate=z, pre_up=u, dgate=dg, dup=du), scalars, element, "silu")
    for a in range(3):
        for b in range(3):
            if a == b:
                continue
            t = [d.clone(), z.clone(), u.clone()]
            launch(kernels.GatedActivationBackward, dict(dout=t[0], pre_gate=t[1], pre_up=t[2], dgate=t[a], dup=t[b]), scalars,
                   element, "silu")
            assert torch.equal(t[a], dg) and torch.equal(t[b], du)


@pytest.mark.parametrize("element", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", IN_PLACE + [(333, 2048), (20, 8200)], ids=str)
def test_in_place_norm_gradients(F, element, kind, shape):
    from triton_metal import _core, kernels
    M, D = shape
    dtype = TYPES[element]
    dn, ds, s, y = (normal(M, D, dtype=dtype) for _ in range(4))
    w, g, p = (normal(D, dtype=dtype, std=0.2, mean=1.0) for _ in range(3))
    stats = torch.rand(M, 4, device="cuda") + 0.5
    scalars = (M, D, _core.float_bits(0.75), D)
    names = ("dnormed", "dsum", "block")

    def run(dresidual, dblock, gate, post, **t):
        sums = [torch.empty_like(w) for _ in range(2)]
        launch(kernels.ResidualNormBackward,
               dict(sum=s, stats=stats, weight=w, gate=gate, post_weight=post, dresidual=dresidual, dblock=dblock,
                    dweight=sums[0], dbias=sums[1], **t), scalars, element, None, kind)
        return sums

    for gate, post in ((None, None), (g, None), (g, p)):
        fresh = dict(zip(names, (dn, ds, y)))
        dr, db = torch.empty_like(s), torch.empty_like(s)
        want = run(dr, db, gate, post, **fresh)
        for a in ("dnormed", "dsum"):
            for b in names:
                if a == b:
                    continue
                t = {k: v.clone() for k, v in fresh.items()}
                got = run(t[a], t[b], gate, post, **t)
                assert torch.equal(t[a], dr) and torch.equal(t[b], db), (a, b)
                assert all(torch.equal(i, j) for i, j in zip(got, want)), (a, b)


@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
def test_in_place_residual_of_every_kernel(F, element):
    dtype = TYPES[element]
    for M, K, N in ((1, 4096, 264), (5, 64, 72), (300, 256, 264), (130, 65, 33), (9486, 136, 792), (1034, 72, 7464), (20, 2, 8)):
        x, w, r = normal(M, K, dtype=dtype), weight(K, N, dtype, "kn"), normal(M, N, dtype=dtype)
        want = F.linear(x, w, None, r, activation="relu")
        assert F.linear(x, w, None, r, activation="relu", out=r) is r and torch.equal(r, want)


# ---- operands the documentation allows ------------------------------------------------------------------------

@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_overlapping_rows_and_shared_operands(F, element):
    """Windows of one signal as rows, one tensor as several operands."""
    dtype = TYPES[element]
    signal = normal(5000, dtype=dtype)
    for K, hop in ((64, 8), (64, 24), (128, 1), (40, 3), (256, 16)):
        x = signal.unfold(0, K, hop)                      # rows hop elements apart
        w = weight(K, 72, dtype, "nk")
        for rows in (x, x[:9], x[:1]):
            assert torch.equal(F.linear(rows, w), F.linear(rows.contiguous(), w))
        d = normal(x.shape[0], 72, dtype=dtype)
        for a, b in zip(F.linear_backward(d, x, w), F.linear_backward(d, x.contiguous(), w)):
            assert a is b is None or torch.equal(a, b)
    for M, K, N in ((7, 64, 72), (140, 65, 33), (300, 128, 264)):
        x, w, d = normal(M, K, dtype=dtype), weight(K, N, dtype, "nk"), normal(M, N, dtype=dtype)
        assert torch.equal(F.gated_linear(x, w, w), F.gated_linear(x, w, w.clone()))
        got, want = F.gated_linear_backward(d, x, w, w, d, d), F.gated_linear_backward(d, x, w, w.clone(), d.clone(), d.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        n = normal(K, dtype=dtype)
        got = F.residual_norm(x, x, n, n, n, n, stats=True)
        assert all(torch.equal(a, b) for a, b in zip(got, F.residual_norm(x, x.clone(), n.clone(), n.clone(), n, n, stats=True)))
        got = F.residual_norm_backward(x, x, x, got[2], n, x, n, n, bias=True)
        want = F.residual_norm_backward(x, x.clone(), x.clone(), F.residual_norm(x, x, n, n, n, n, stats=True)[2], n, x.clone(),
                                        n.clone(), n.clone(), bias=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
def test_extents_of_zero(F, element):
    dtype = TYPES[element]
    new = lambda *s: normal(*s, dtype=dtype)  # noqa: E731
    for M, K, N in ((0, 16, 24), (5, 0, 24), (5, 16, 0), (0, 0, 0), (1, 0, 1)):
        x, w, d, b = new(M, K), new(K, N), new(M, N), new(N)
        out, pre = F.linear(x, w, b, d, activation="sigmoid", pre=True)
        assert torch.equal(pre, b.expand(M, N)) or K
        if not K:
            error = (out.double() - (torch.sigmoid(b.double()) + d.double())).abs()
            assert not error.numel() or float(error.max()) <= 8 * half(dtype)
        dx, dw, db = F.linear_backward(d, x, w, d, activation="silu", bias=True)
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        assert not (dw != 0).any() and (N or not (dx != 0).any()) and (M or not (db != 0).any())
        h, g, u = F.gated_linear(x, w, w, save=True)
        assert h.shape == (M, N) and (K or not ((h != 0) | (g != 0) | (u != 0)).any())
        dx, dwg, dwu = F.gated_linear_backward(d, x, w, w, g, u)
        assert not ((dwg != 0) | (dwu != 0)).any() and (N or not (dx != 0).any())
    total, normed, stats = F.residual_norm(new(0, 64), new(0, 64), new(64), stats=True)
    back = F.residual_norm_backward(normed, total, total, stats, new(64), total, new(64), new(64), bias=True)
    assert total.shape == normed.shape == (0, 64) and stats.shape == (0, 4)
    assert all(not (v != 0).any() for v in back)


@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_one_row_without_a_batch_dimension(F, element):
    dtype = TYPES[element]
    x, w, n, d = normal(264, dtype=dtype), weight(264, 72, dtype, "kn"), normal(264, dtype=dtype), normal(72, dtype=dtype)
    one = lambda t: t.unsqueeze(0)  # noqa: E731
    assert torch.equal(one(F.linear(x, w, None, d)), F.linear(one(x), w, None, one(d)))
    for a, b in zip(F.linear_backward(d, x, w), F.linear_backward(one(d), one(x), w)):
        assert a is b is None or torch.equal(a, b.view(a.shape))
    assert torch.equal(one(F.gated_linear(x, w, w)), F.gated_linear(one(x), w, w))
    s, m, st = F.residual_norm(x, x, n, stats=True)
    wanted = F.residual_norm(one(x), one(x), n, stats=True)
    assert s.shape == m.shape == x.shape and all(torch.equal(a.view(b.shape), b) for a, b in zip((s, m, st), wanted))
    got = F.residual_norm_backward(m, s, s, st, n, x)
    assert got[0].shape == got[1].shape == x.shape


# ---- operands of more than 2^31 elements --------------------------------------------------------------------

FAR = 5                                    # rows at the far end that hold something


def far(M, N, dtype):
    """Zeros, but for the first and the last few rows."""
    t = torch.zeros(M, N, device="cuda", dtype=dtype)
    assert t.numel() > 1 << 31
    for rows in (t[:FAR], t[-FAR:]):
        rows.copy_(normal(FAR, N, dtype=dtype))
    return t


def test_far_rows_of_the_norms_and_activation_gradients(F):
    dtype, M, D = torch.bfloat16, 140000, 16384
    w, g, p = (normal(D, dtype=dtype, std=0.1, mean=1.0) for _ in range(3))
    r, y = far(M, D, dtype), far(M, D, dtype)
    ends = lambda *ts: [torch.cat([t[:FAR], t[-FAR:]]) for t in ts]  # noqa: E731
    total, normed, stats = F.residual_norm(r, y, w, w, g, p, kind="layer", stats=True)
    want = F.residual_norm(*ends(r, y), w, w, g, p, kind="layer", stats=True)
    assert all(torch.equal(a, b) for a, b in zip(ends(total, normed, stats), want))
    del normed, r
    dn = far(M, D, dtype)
    got = F.residual_norm_backward(dn, None, total, stats, w, y, g, p, kind="layer")[:2]
    back = F.residual_norm_backward(*ends(dn), None, *ends(total, stats), w, *ends(y), g, p, kind="layer")
    assert all(torch.equal(a, b) for a, b in zip(ends(*got), back))
    del got, total
    one = weight(8, D, dtype, "kn")
    x = torch.zeros(M, 8, device="cuda", dtype=dtype)
    dx, _, db = F.linear_backward(dn, x, one, y, activation="silu", bias=True)       # dz of 2^31 elements and more
    few = F.linear_backward(*ends(dn, x), one, *ends(y), activation="silu", bias=True)
    scale = float(few[0].double().abs().max())
    assert float((ends(dx)[0].double() - few[0].double()).abs().max()) < 2 * half(dtype) * scale
    assert not (dx[FAR:-FAR] != 0).any()
    assert float((db.double() - few[2].double()).abs().max()) < 2 * half(dtype) * float(few[2].double().abs().max())


@pytest.mark.parametrize("element", ["bf16", "f32"])
def test_far_columns_of_weights_and_rows_of_outputs(F, element):
    """Weights of more than 2^31 elements (aligned, and at an odd pitch, which are copied first), then outputs."""
    dtype = TYPES[element]
    for K, N in ((70000, 32768),) + (((70001, 32765),) if element == "bf16" else ()):
        w = torch.zeros(K, N, device="cuda", dtype=dtype)
        w[-64:].copy_(normal(64, N, dtype=dtype, std=0.125))
        for M in (3, 200):
            x = normal(M, K, dtype=dtype)
            z, slack = product64(x[:, -64:], w[-64:])
            check(F.linear(x, w), z, slack)
        del w
    for K, N in ((64, 32768), (2, 32769)):
        M = 70000
        x, w = normal(M, K, dtype=dtype), weight(K, N, dtype, "kn")
        out = F.linear(x, w)
        for rows in (slice(0, 9), slice(M - 9, M)):
            z, slack = product64(x[rows], w)
            check(out[rows], z, slack)
        del out
    torch.cuda.empty_cache()


def test_the_widest_products_on_the_cuda_cores(F):
    """The last size that is taken is right to its last column, and the refusal of the next names the limit."""
    for columns, call in ((8388480, lambda x, w: F.linear(x, w)), (4194240, lambda x, w: F.gated_linear(x, w, w, activation="none"))):
        x, w = normal(2, 3, dtype=torch.float32), normal(3, columns + 1, dtype=torch.float32)
        z, slack = product64(x, w[:, :columns])
        got = call(x, w[:, :columns])
        if columns == 8388480:
            check(got, z, slack)
        else:
            check(got, z * z, slack * (2 * z.abs() + slack) + 2.0 ** -23 * z * z)
        with pytest.raises(RuntimeError, match=f"more than {columns} columns"):
            call(x, w)


def test_products_that_take_longer_than_a_wait_may(F):
    """Sums so long that a tile takes about as long as the bounded waits' second, or longer: nothing gives up."""
    dtype, at = torch.bfloat16, [0, 1, 77, 1 << 28, (1 << 29) - 3]
    # few rows: one row, one column, K of almost 2^31
    K = (1 << 31) - 600
    x, w = torch.zeros(1, K, device="cuda", dtype=dtype), torch.zeros(K, 1, device="cuda", dtype=dtype)
    far_at = torch.tensor(at + [K - 1, K // 2], device="cuda")
    x[0, far_at], w[far_at, 0] = normal(far_at.numel(), dtype=dtype), normal(far_at.numel(), dtype=dtype)
    z, slack = product64(x[:, far_at], w[far_at])
    check(F.linear(x, w), z, slack)
    nothing_gave_up(F)
    del x, w
    # the CTA pairs: the gradient of a 2 x 2 weight over 2^29 rows
    M = 1 << 29
    x, d, w = torch.zeros(M, 2, device="cuda", dtype=dtype), torch.zeros(M, 2, device="cuda", dtype=dtype), weight(2, 2, dtype, "kn")
    rows = torch.tensor(at, device="cuda")
    x[rows], d[rows] = normal(len(at), 2, dtype=dtype), normal(len(at), 2, dtype=dtype)
    dx, dw, _ = F.linear_backward(d, x, w)
    nothing_gave_up(F)
    z, slack = product64(x[rows].t(), d[rows])
    check(dw, z, slack)
    z, slack = product64(d[rows], w.t())
    check(dx[rows], z, slack)
    del x, d, dx
    torch.cuda.empty_cache()


def nothing_gave_up(F):
    torch.cuda.synchronize()
    F.check()
