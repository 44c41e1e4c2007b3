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


@pytest.mark.parametrize("name", ["gz_adamw_get_steps", "gz_adamw_set_steps"])
def test_entry_points_are_declared(name):
    from pathlib import Path

    assert name in (Path(gz.__file__).resolve().parents[1] / "include" / "graphzero_b200.h").read_text()
