"""CPU-side checks of the operators on logits: the binding's structs have the header's layout,
bfloat16 conversions round as they say, and a null context is refused."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("c_name,py_name", [("pcu_logits", "Logits"), ("pcu_distill", "Distill"), ("pcu_sampling", "Sampling")])
def test_structs_have_the_headers_layout(pcu_pkg, c_name, py_name):
    from fusion_pcu_amd import _abi
    fields = [f for f, _ in getattr(_abi, py_name)._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "pcu_rocm.h"\nint main(void){printf("%zu", sizeof(' + c_name + "));"
    for f in fields:
        src += f'printf(" %zu", offsetof({c_name}, {f}));'
    src += "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "layout.c")
        with open(path, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), path, "-o", os.path.join(d, "layout")], check=True)
        out = subprocess.run([os.path.join(d, "layout")], capture_output=True, text=True, check=True).stdout
    mirror = getattr(_abi, py_name)
    assert [int(v) for v in out.split()] == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


def test_bfloat16_rounds_to_nearest_even(pcu_pkg):
    rng = np.random.default_rng(0)
    bits = rng.integers(0, 2 ** 32, 200000, dtype=np.uint64).astype(np.uint32)
    ties = (rng.integers(0, 2 ** 16, 5000).astype(np.uint32) << 16) | 0x8000
    x = np.concatenate([bits, ties, np.array([0, 0x80000000, 0x7F800000, 0xFF800000, 1, 0x7F7FFFFF], np.uint32)]).view(np.float32)
    got = pcu_pkg.from_bfloat16(pcu_pkg.to_bfloat16(x))
    assert np.array_equal(np.isnan(got), np.isnan(x))
    keep = ~np.isnan(x)
    x, got = x[keep], got[keep]
    # The two neighbours with 8 significant bits, and the nearer of them (the even one of a tie).
    low = (x.view(np.uint32) & np.uint32(0xFFFF0000))
    high = (low.astype(np.uint64) + 0x10000).astype(np.uint32)
    rest = x.view(np.uint32) & np.uint32(0xFFFF)
    up = (rest > 0x8000) | ((rest == 0x8000) & ((low >> 16) & 1 == 1))
    want = np.where(np.isinf(x) | ~up, low, high)
    assert np.array_equal(got.view(np.uint32), want)
    stored = pcu_pkg.to_bfloat16(np.float32(got))
    assert np.array_equal(pcu_pkg.from_bfloat16(stored).view(np.uint32), got.view(np.uint32))


def test_a_null_context_is_refused(pcu_pkg):
    from fusion_pcu_amd import _abi
    lib = pcu_pkg.lib()
    lg, d, p = _abi.Logits(), _abi.Distill(), _abi.Sampling()
    lg_p, d_p, p_p = ctypes.byref(lg), ctypes.byref(d), ctypes.byref(p)
    assert lib.pcu_native_top_logits(None, lg_p, 1, 1.0, None, None, None) == _abi.PCU_ERR_ARGUMENT
    assert lib.pcu_native_distill_loss(None, lg_p, d_p, None, None, None) == _abi.PCU_ERR_ARGUMENT
    assert lib.pcu_native_distill_backward(None, lg_p, d_p, None, None, None, 0, 0, None) == _abi.PCU_ERR_ARGUMENT
    assert lib.pcu_native_distill_step(None, lg_p, d_p, None, None, None, 0, 0, None) == _abi.PCU_ERR_ARGUMENT
    assert lib.pcu_native_sample(None, lg_p, p_p, None, None, None) == _abi.PCU_ERR_ARGUMENT


@pytest.mark.parametrize("top_k,passed", [(5, 5), (0, 0), (-3, -1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 0),
                                          (2 ** 32 + 5, 0), (-2 ** 32 + 7, 0), (np.int64(2 ** 40), 0), (np.int32(7), 7)])
def test_a_top_k_beyond_32_bits_sets_no_limit(pcu_pkg, top_k, passed):
    """The C ABI takes 32 bits; a larger number is no limit (0), not what its low bits say."""
    from fusion_pcu_amd import _abi
    seen = []

    class Lib:
        def pcu_native_sample(self, handle, logits, sampling, tokens, log_prob, fault):
            seen.append(sampling._obj.top_k_value)
            return _abi.PCU_OK

    ctx = pcu_pkg.Context.__new__(pcu_pkg.Context)
    ctx.handle, ctx._lib = None, Lib()
    array = lambda shape, dtype: pcu_pkg.DeviceArray(ctx, 4096, shape, dtype)
    ctx.native_sample(array((2, 9), np.float32), array((2,), np.float32), top_k=top_k,
                      tokens=array((2,), np.int32), log_prob=array((2,), np.float32))
    assert seen[0] == passed or (seen[0] <= 0 and passed <= 0)
    with pytest.raises(TypeError):
        ctx.native_sample(array((2, 9), np.float32), array((2,), np.float32), top_k=2.5,
                          tokens=array((2,), np.int32), log_prob=array((2,), np.float32))
