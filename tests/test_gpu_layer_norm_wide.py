"""Layer norm's gradients of rows too long to hold in registers, each of them alone, on the GPU: the bits of the call that
computes all, and no more scratch than they need. And the statistics of rows without columns."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype,code", [(np.float32, 0), (np.float64, 1), (np.float16, 3)])
@pytest.mark.parametrize("rows,width", [(1, 16385), (3, 20001), (300, 17000)])
def test_each_gradient_alone(ctx, rows, width, dtype, code):
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(rows)
    x, dy, w = (ctx.upload(rng.normal(0, 1, s).astype(dtype)) for s in ((rows, width), (rows, width), (width,)))
    _, stats = ctx.native_layer_norm(x, w)
    whole = [a.numpy() for a in ctx.native_layer_norm_backward(x, stats, dy, w)]
    rows_of = ctypes.byref(_abi.Rows(x.ptr, code, 0, rows, width, width))
    for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1), (0, 0, 0)):
        out = [ctx.upload(np.full(s, 3, dtype)) for s in ((rows, width), (width,), (width,))]
        ptrs = [a.ptr if on else None for a, on in zip(out, want)]
        assert ctx._lib.pcu_native_layer_norm_backward(ctx.handle, rows_of, stats.ptr, dy.ptr, width, w.ptr, code, ptrs[0], width,
                                                       ptrs[1], ptrs[2]) == 0
        for a, b, on in zip(out, whole, want):
            np.testing.assert_array_equal(a.numpy(), b if on else np.full_like(b, 3))


def _pool_bytes():
    """What is in use of the device's memory pool (hipMemPoolAttrUsedMemCurrent), by the runtime that the library loaded."""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip, pool, used = ctypes.CDLL(path), ctypes.c_void_p(), ctypes.c_uint64()
    assert hip.hipDeviceGetDefaultMemPool(ctypes.byref(pool), 0) == 0
    assert hip.hipMemPoolGetAttribute(pool, 7, ctypes.byref(used)) == 0
    return used.value


def test_the_rows_gradient_alone_takes_no_columns_sums(pcu_pkg):
    """256 rows of 131072 binary64 values: the columns' sums of 256 workgroups are 512 MiB of scratch."""
    rows, width = 256, 1 << 17
    with pcu_pkg.Context(0) as c:
        x, dy, dx = (c.empty((rows, width), np.float64) for _ in range(3))
        _, stats = c.native_layer_norm(x, out=dx)
        before = _pool_bytes()
        c.native_layer_norm_backward(x, stats, dy, x_gradient=dx)
        assert _pool_bytes() - before < 1 << 20
        c.native_layer_norm_backward(x, stats, dy, x_gradient=dx, weight_gradient=c.empty((width,), np.float64))
        assert _pool_bytes() - before >= 512 << 20


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
@pytest.mark.parametrize("rows", [1, 3000])
def test_statistics_of_no_columns(ctx, rows, dtype):
    """The mean of nothing is 0 / 0."""
    stats = ctx.upload(np.full((rows, 2), 3, np.float64 if dtype == np.float64 else np.float32))
    out, _ = ctx.native_layer_norm(ctx.empty((rows, 0), dtype), stats=stats)
    assert out.shape == (rows, 0) and np.all(np.isnan(stats.numpy()))
