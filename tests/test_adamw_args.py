"""Refusals of AdamW's entry points that come before any GPU call."""
import ctypes as C

import pytest

import graphzero_b200 as gz

L = gz._lib


def test_step_counts():
    n = C.c_int64(5)
    assert L.gz_adamw_get_steps(None, C.byref(n)) == gz.ERR_INVALID_ARG and n.value == 5
    assert L.gz_adamw_set_steps(None, 3) == gz.ERR_INVALID_ARG
    assert b"gz_adamw_set_steps" in L.gz_last_error()


def plan(bits, *tensors):
    h = C.c_void_p()
    status = L.gz_adamw_create((gz.AdamWTensor * len(tensors))(*tensors), len(tensors), bits, -1, C.byref(h))
    assert not h
    return status, L.gz_last_error()


def tensor(at, n, **kw):
    far = at * 16
    return gz.AdamWTensor(**(dict(param=at, copy=None, m=far, v=far + 0x100000, m_scale=far + 0x200000, v_scale=far + 0x300000, n=n,
                                  weight_decay=0.0, lr_scale=1.0, copy_dtype=gz.BF16) | kw))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("a,b", [
    (dict(), dict(param=0x1000)),                              # a weight twice
    (dict(), dict(param=0x1000 + 4 * 299)),                    # the last of the first
    (dict(), dict(param=0x1000 - 4 * 299)),
    (dict(), dict(m=0x10000)), (dict(), dict(v=0x10000)), (dict(v=0x10000), dict()),
    (dict(copy=0x700000), dict(copy=0x700000 + 2 * 299)), (dict(copy=0x1000 + 4 * 150), dict()),
], ids=str)
def test_overlapping_buffers(a, b, bits):
    """Blocks of threads would race for what two tensors share (no device is needed to refuse it)."""
    status, message = plan(bits, tensor(0x1000, 300, **a), tensor(0x40000, 300, **b))
    assert status == gz.ERR_INVALID_ARG and b"overlap" in message


def test_scales_and_the_rounded_up_end_of_8bit_states():
    for kw in (dict(m_scale=0x10000 + 0x300000), dict(v_scale=0x10000 + 0x200004), dict(m=0x10000 + 496)):
        status, message = plan(8, tensor(0x1000, 300), tensor(0x40000, 300, **kw))
        assert status == gz.ERR_INVALID_ARG and b"overlap" in message
    status, message = plan(32, tensor(0x1000, 300), tensor(0x40000, 300, m_scale=0x1000))  # unused with 32 bits
    assert b"overlap" not in message


def test_neighbours_do_not_overlap():
    for bits in (8, 32):
        status, message = plan(bits, tensor(0x1000, 300), tensor(0x1000 + 4 * 300, 300, m=0x20000, v=0x800000, m_scale=0x900000,
                                                                 v_scale=0xa00000), tensor(0x1000, 0))
        assert status != gz.OK and b"overlap" not in message  # (there is no device -1)


@pytest.mark.parametrize("name", ["gz_adamw_get_steps", "gz_adamw_set_steps"])
def test_entry_points_are_declared(name):
    from pathlib import Path

    assert name in (Path(gz.__file__).resolve().parents[1] / "include" / "graphzero_b200.h").read_text()
