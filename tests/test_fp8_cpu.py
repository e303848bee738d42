"""The FP8 and balance entry points where no GPU is needed: refusals without a context, and the 64-bit reference itself."""
import numpy as np

import fp8_ref as ref


def test_null_arguments_are_refused(pkg):
    lib = pkg.load_library()
    assert lib.qkm_fp8_quantize(None, None, 1, 128, None, None) == -1
    assert lib.qkm_fp8_gemm(None, None, None, None, None, None, 16, 128, 1) == -1
    assert lib.qkm_moe_gateup_grouped_fp8(None, *[None] * 9, 1) == -1
    assert lib.qkm_moe_down_grouped_fp8(None, *[None] * 8, 1) == -1
    assert lib.qkm_moe_shared_gateup_fp8(None, *[None] * 7, 1) == -1
    assert lib.qkm_moe_shared_down_fp8(None, *[None] * 6, 1) == -1
    assert lib.qkm_moe_balance(None, None, None, None, 1, 1.0, None, None, None) == -1
    assert lib.qkm_moe_balance_grad(None, None, None, None, 1, 1.0, None, None) == -1


def test_fast_calls_convert_like_ctypes(pkg):
    """The extension module's forms reach the library (which refuses the NULL context) and refuse a wrong number of arguments."""
    import pytest
    ctx = object.__new__(pkg.Context)
    ctx.lib, ctx.h = pkg.load_library(), None
    from qwen_kernel_b200 import qkm_calls
    ctx._calls = qkm_calls
    for call in (lambda: ctx.fp8_quantize(None, 1, 128, 0, 0), lambda: ctx.fp8_gemm(0, 0, 0, 0, 0, 16, 128, 1),
                 lambda: ctx.moe_balance(0, 0, None, 1, 0.5, 0, 0, 0), lambda: ctx.moe_balance_grad(0, None, 0, 1, 1e-2, None, 0)):
        with pytest.raises(pkg.QkmError) as ei:
            call()
        assert ei.value.code == -1
    with pytest.raises(TypeError):
        qkm_calls.fp8_gemm(None, 0, 0)


def test_reference_codes():
    """Every code comes back from its value; halves go to the even code."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(ref.encode(ref.decode(codes)), codes)
    v = ref.decode(np.arange(127))
    mid = (v[1:] + v[:-1]) / 2
    got = ref.encode(mid)
    assert np.all(got % 2 == 0) and np.all(np.abs(got.astype(int) - np.arange(126) - 0.5) == 0.5)
    q, s = ref.quantize(np.array([[448.0] + [0.0] * 15, [448.1] + [1.0] * 15, [0.0] * 16, [1e-45] + [0.0] * 15], np.float32))
    assert s.ravel().tolist() == [1.0, 2.0, 1.0, 2.0**-126] and q[0, 0] == 126 and not q[2].any()
