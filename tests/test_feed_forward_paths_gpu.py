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
