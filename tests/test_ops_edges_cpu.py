"""The operators' edges that need no GPU: refusals, verdicts and sizes."""
import pytest

import zepp_b200 as zb
from zepp_b200 import ops
from zepp_b200._ext import lib


def error(rc):
    assert rc != 0
    return lib().zepp_last_error().decode()


def test_wait_limit():
    assert "wait limit" in error(ops._fn("zepp_op_set_wait_limit_ns")(-1))
    for bad in (-1.0, float("nan"), float("inf"), 3601):
        with pytest.raises(AssertionError):
            ops.set_wait_limit(bad)
    ops.set_wait_limit(2)
