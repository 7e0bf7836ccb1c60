"""CPU checks of the 4-bit key / value cache: the header, the library's exports and what needs no GPU."""
import ctypes

import numpy as np
import pytest

import cache4_lib as C
import we


def test_every_declared_function_is_exported_and_bound():
    declared = we.header_functions(we.CACHE4_HEADER)
    assert set(declared) == set(we.CACHE4_SIGNATURES) and len(declared) == 5
    lib = we.load_library()
    assert all(hasattr(lib, name) for name in declared)


@pytest.mark.parametrize("shape,bytes_,message", [
    ((1, 1, 64, 64), 64 * 72, None), ((3, 5, 256, 128), 3 * 5 * 128 * 288, None),
    ((65535, 1, 128, 1 << 24), 65535 * (1 << 24) * 144, None),
    ((1, 1, 0, 64), 0, "dim must be a multiple of 64 and at most 256, got 0"), ((1, 1, 100, 64), 0, "got 100"),
    ((1, 1, 512, 64), 0, "got 512"), ((1, 1, 64, 0), 0, "capacity must be a multiple of 64"),
    ((1, 1, 64, (1 << 24) + 64), 0, "capacity must be"), ((0, 1, 64, 64), 0, "batch and kvHeads"),
    ((1, 70000, 64, 64), 0, "batch and kvHeads"),
])
def test_bytes(shape, bytes_, message):
    lib, c, n = we.load_library(), we.Cache4Struct(*shape, None), ctypes.c_uint64()
    rc = lib.we_cache4_bytes(None, ctypes.byref(c), ctypes.byref(n))
    if message is None:
        assert rc == 0 and n.value == bytes_
    else:
        assert rc and message in lib.we_last_error(None).decode()


def test_calls_without_a_context_are_refused():
    lib, c = we.load_library(), we.Cache4Struct(1, 1, 64, 64, None)
    for name, (_, args) in we.CACHE4_SIGNATURES.items():
        if name != "we_cache4_bytes":
            assert getattr(lib, name)(*[None if a is ctypes.c_void_p else 0 for a in args]) == we.WE_EINVAL
            assert "context is null" in lib.we_last_error(None).decode()
    assert lib.we_cache4_bytes(None, ctypes.byref(c), None) == we.WE_EINVAL
    assert lib.we_cache4_bytes(None, None, ctypes.byref(ctypes.c_uint64())) == we.WE_EINVAL


def test_plain_form_rounds_to_the_nearest_code():
    """the oracle itself: a stored value is at most half a step off, and by what its scale and minimum round off"""
    x = np.random.default_rng(0).standard_normal((5, 3, 192)).astype(np.float32).astype(np.float64)
    codes, scales = C.quantize(x)
    y = C.dequantize(codes, scales)
    s = (scales & 0xffff).astype(np.uint16).view(np.float16).astype(np.float64).repeat(64, -1)
    # code 15 reaches the maximum but for the roundings of the scale (15 half steps) and of the minimum
    assert (np.abs(y - x) <= s * (0.5 + 15 * 2.0 ** -11) + np.abs(x).max() * 2.0 ** -11 + 1e-7).all()
