"""A bounded wait that gave up reaches callers who never synchronise through the library.  The record is written from
the host (tmx_debug_inject_status), as a kernel would write it."""

import pytest

torch = pytest.importorskip("torch")

from tmtest import require_gpu  # noqa: E402

pytestmark = pytest.mark.gpu


def test_the_next_call_reports_it_once(core):
    require_gpu()
    from triton_metal import cuda, functional as F
    x, w, n = torch.randn(4, 64, device="cuda"), torch.randn(64, 32, device="cuda"), torch.ones(64, device="cuda")
    try:
        want = F.linear(x, w)
        cuda.inject_status(1, 53, 7, 0)
        launches = cuda.launch_count()
        with pytest.raises(RuntimeError, match=r"gave up inside the kernel \(code 1, site 53, block 7.*an earlier launch"):
            F.linear(x, w)
        assert cuda.launch_count() == launches
        assert torch.equal(F.linear(x, w), want)
        cuda.inject_status(1, 61, 0, 0)
        with pytest.raises(RuntimeError, match="site 61"):
            F.residual_norm(x, None, n)
        F.residual_norm(x, None, n)
        # without another launch, and without a wait of the library's
        F.check()
        cuda.inject_status(1, 54, 0, 0)
        with pytest.raises(RuntimeError, match="site 54.*an earlier launch are not valid"):
            F.check()
        F.check()
        assert torch.equal(F.linear(x, w), want)
    finally:
        F.release()


def test_a_refused_call_leaves_the_record(core):
    require_gpu()
    from triton_metal import cuda, functional as F
    x, w = torch.randn(16, 16, device="cuda"), torch.randn(16, 16, device="cuda")
    try:
        cuda.inject_status(1, 42, 0, 0)
        with pytest.raises(RuntimeError, match="out overlaps its input x"):
            F.linear(x, w, out=x)
        with pytest.raises(RuntimeError, match="site 42"):
            F.check()
    finally:
        F.check()
        F.release()
