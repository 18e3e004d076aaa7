"""CPU-side checks of the operators around a model's products: the binding's struct has the header's
layout, a null context is refused, and arguments are checked before any pointer reaches the library."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_have_the_headers_layout(pcu_pkg):
    from fusion_pcu_amd import _abi
    fields = [f for f, _ in _abi.Rows._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "pcu_rocm.h"\nint main(void){printf("%zu", sizeof(pcu_rows));'
    for f in fields:
        src += f'printf(" %zu", offsetof(pcu_rows, {f}));'
    src += "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "layout.c")
        with open(path, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), path, "-o", os.path.join(d, "layout")], check=True)
        out = subprocess.run([os.path.join(d, "layout")], capture_output=True, text=True, check=True).stdout
    assert [int(v) for v in out.split()] == [ctypes.sizeof(_abi.Rows)] + [getattr(_abi.Rows, f).offset for f in fields]


def test_a_null_context_is_refused(pcu_pkg):
    from fusion_pcu_amd import _abi
    lib, r = pcu_pkg.lib(), ctypes.byref(_abi.Rows())
    bad = _abi.PCU_ERR_ARGUMENT
    assert lib.pcu_native_embedding(None, r, None, 0, 1.0, None, 0, None) == bad
    assert lib.pcu_native_embedding_backward(None, r, None, 0, 1.0, None, 0, None, 0, None) == bad
    assert lib.pcu_native_layer_norm(None, r, None, None, 0, 1e-5, None, 0, None) == bad
    assert lib.pcu_native_layer_norm_backward(None, r, None, None, 0, None, 0, None, 0, None, None) == bad


class _NoCalls:
    """A library that nothing may call."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture()
def ctx(pcu_pkg):
    c = pcu_pkg.Context.__new__(pcu_pkg.Context)
    c.handle, c._lib = None, _NoCalls()
    return c


def test_shapes_and_types_are_checked_first(ctx, pcu_pkg):
    array = lambda shape, dtype=np.float32: pcu_pkg.DeviceArray(ctx, 4096, shape, dtype)
    table, tokens, x, stats = array((10, 8)), array((4,), np.int32), array((4, 8)), array((4, 2))
    for call in (lambda: ctx.native_embedding(array((10,)), tokens), lambda: ctx.native_embedding(table, array((4,))),
                 lambda: ctx.native_embedding(table, array((2, 2), np.int32)), lambda: ctx.native_embedding(table, tokens, out=array((4, 9))),
                 lambda: ctx.native_embedding(table, tokens, out=array((4, 8), np.float16)),
                 lambda: ctx.native_embedding(array((10, 8), np.int64), tokens),
                 lambda: ctx.native_embedding_backward(x, array((5,), np.int32), 10),
                 lambda: ctx.native_embedding_backward(x, tokens, -1), lambda: ctx.native_embedding_backward(x, tokens, 1 << 23),
                 lambda: ctx.native_embedding_backward(x, tokens, 10, base=array((10, 8), np.float64), out=table),
                 lambda: ctx.native_embedding_backward(x, tokens, 10, out=array((11, 8))),
                 lambda: ctx.native_layer_norm(array((8,)), out=x, stats=stats), lambda: ctx.native_layer_norm(x, array((9,)), out=x, stats=stats),
                 lambda: ctx.native_layer_norm(x, array((8,), np.float16), out=x, stats=stats),
                 lambda: ctx.native_layer_norm(x, array((8,)), array((8,), np.float64), out=x, stats=stats),
                 lambda: ctx.native_layer_norm(x, out=array((4, 8), np.float64), stats=stats),
                 lambda: ctx.native_layer_norm(x, out=x, stats=array((4, 2), np.float64)),
                 lambda: ctx.native_layer_norm_backward(x, array((4,)), x), lambda: ctx.native_layer_norm_backward(x, stats, array((4, 7))),
                 lambda: ctx.native_layer_norm_backward(x, stats, x, x_gradient=array((3, 8))),
                 lambda: ctx.native_layer_norm_backward(x, stats, x, array((8,)), x_gradient=x, weight_gradient=array((7,)))):
        with pytest.raises(pcu_pkg.PcuExecutionError):
            call()
    with pytest.raises(TypeError):
        ctx.native_embedding_backward(x, tokens, 10.5)
