"""The paged cache's descriptions, without a device: what is refused, and what a plan takes."""
import ctypes as C

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200 import _lib
from lapid_b200.paged import Mask, PagedSpec, plan_bytes, rope_table

OK = dict(dtype=lp.DType.BF16, q_heads=32, kv_heads=8, head_dim=128, page_size=16, pages=1000, requests=4, tokens=40, max_blocks=64, max_new=10)


@pytest.mark.parametrize("change,code", [
    ({"dtype": lp.DType.F32}, "unsupported_dtype"), ({"dtype": lp.DType.Q4K}, "unsupported_dtype"), ({"q_heads": 30}, "invalid_launch"), ({"kv_heads": 0}, "invalid_launch"),
    ({"q_heads": 0}, "invalid_launch"), ({"head_dim": 12}, "unsupported"), ({"head_dim": 8}, "unsupported"), ({"head_dim": 136}, "unsupported"), ({"head_dim": 100}, "unsupported"),
    ({"page_size": 8}, "unsupported"), ({"page_size": 48}, "unsupported"), ({"page_size": 256}, "unsupported"), ({"pages": 0}, "invalid_launch"), ({"pages": 1 << 28}, "too_large"),
    ({"pages": 1 << 62}, "too_large"), ({"requests": 1 << 31}, "too_large"), ({"requests": 1 << 26}, "too_large"), ({"tokens": 1 << 27}, "too_large"), ({"max_blocks": 1 << 29}, "too_large"),
    ({"max_blocks": 1 << 23, "tokens": 1 << 16}, "too_large"), ({"max_new": 1 << 30}, "too_large"), ({"mask": 3}, "invalid_argument"), ({"mask": Mask.FULL, "window": 5}, "invalid_argument"),
    ({"window": 1 << 31}, "too_large"), ({"scale": float("nan")}, "invalid_argument"), ({"scale": float("inf")}, "invalid_argument"), ({"tokens": -1}, "invalid_argument")])
def test_descriptions_that_are_refused(change, code):
    with pytest.raises(lp.LapidError) as e:
        plan_bytes(PagedSpec(**{**OK, **change}))
    assert e.value.code == code


def test_plan_bytes_grow_with_what_is_planned():
    few, many = plan_bytes(PagedSpec(**{**OK, "max_new": 1})), plan_bytes(PagedSpec(**{**OK, "max_new": 100}))
    assert 0 < few < 8 << 20 and few < many < 64 << 20
    assert plan_bytes(PagedSpec(**{**OK, "requests": 0, "tokens": 0})) > 0
    n = C.c_uint64(7)
    assert _lib.lib().lapid_b200_paged_plan_bytes(None, C.byref(n)) == 1 and n.value == 7
    assert C.sizeof(_lib.PagedC) == 80 and _lib.PagedC.pages.offset == 24 and _lib.PagedC.scale.offset == 72


def test_null_device_is_refused():
    c = PagedSpec(**OK).to_c()
    lib = _lib.lib()
    assert lib.lapid_b200_paged_plan(None, C.byref(c), *[None] * 3, 0, *[None] * 6) == 1
    assert lib.lapid_b200_paged_attention(None, C.byref(c), *[None] * 9) == 1
    assert lib.lapid_b200_paged_append(None, C.byref(c), 0, *[None] * 7, 0, 0, 0, *[None] * 5) == 1


def test_rope_table():
    t = rope_table(10, 8)
    assert t.shape == (10, 8) and t.dtype == np.float32
    assert np.allclose(t[3], np.concatenate([np.cos(3.0 * 10000.0 ** (-np.arange(4) / 4)), np.sin(3.0 * 10000.0 ** (-np.arange(4) / 4))]), atol=1e-7)
