"""The operators' refusals and the layouts of their arguments: nothing here needs a GPU."""
import ctypes

import pytest
import torch

import zepp_b200 as zb
from zepp_b200 import ops
from zepp_b200._ext import lib


def test_public_names():
    for name in ("route_topk", "sort_tokens", "unsort_tokens", "SortPlan", "expert_ffn", "grad_norm", "clip_grad_norm_"):
        assert name in zb.__all__ and getattr(zb, name) is getattr(ops, name)
    for name in ops._ARGS:
        assert hasattr(lib(), name)


@pytest.mark.parametrize("call", [
    lambda: ops.route_topk(torch.zeros(4, 8), 2),                                     # not on a GPU
    lambda: ops.sort_tokens(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), 4),
    lambda: ops.unsort_tokens(torch.zeros(8, 8), ops.SortPlan(torch.zeros(5, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32))),
    lambda: ops.expert_ffn(torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 16, 8), torch.zeros(2, 8, 8)),
    lambda: ops.expert_ffn(torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 16, 8), torch.zeros(2, 8, 8), act="relu"),
    lambda: ops.grad_norm([]),
    lambda: ops.grad_norm([torch.zeros(3)]),
    lambda: ops.clip_grad_norm_([torch.zeros(3)], -1.0),
    lambda: ops.clip_grad_norm_([torch.zeros(3)], float("nan")),
])
def test_refusals_without_a_gpu(call):
    with pytest.raises(AssertionError):
        call()


def _error(rc):
    assert rc != 0
    return lib().zepp_last_error().decode()


def test_c_entry_points_refuse_before_any_gpu_call():
    f = ops._fn
    assert "element type" in _error(f("zepp_op_gate")(None, 7, 1, 8, 2, 0, 1, None, 1.0, None, None, None))
    assert "experts" in _error(f("zepp_op_gate")(None, 0, 1, 1025, 2, 0, 1, None, 1.0, None, None, None))
    assert "top-k" in _error(f("zepp_op_gate")(None, 0, 1, 8, 9, 0, 1, None, 1.0, None, None, None))
    assert "top-k" in _error(f("zepp_op_gate")(None, 0, 1, 64, 33, 0, 1, None, 1.0, None, None, None))
    assert "sigmoid" in _error(f("zepp_op_gate")(None, 0, 1, 8, 2, 0, 1, 16, 1.0, None, None, None))
    assert "tokens" in _error(f("zepp_op_gate_grad")(None, 0, -1, 8, 2, 0, 1, 1.0, None, None, None, None, None))
    assert "top-k" in _error(f("zepp_op_sort")(None, 0, 1, 65, 8, None, None, 0, 8, None, None, None, None, None))
    assert "experts" in _error(f("zepp_op_sort")(None, 0, 1, 2, 8, None, None, 0, 2049, None, None, None, None, None))
    assert "32-bit" in _error(f("zepp_op_unsort")(None, 0, 1 << 30, 2, 8, None, None, None, None))
    assert "elements" in _error(f("zepp_op_unsort_grad")(None, None, 0, 4, 2, 0, 8, None, None, None, None, None, None))
    ffn = f("zepp_op_expert_ffn")
    assert "multiples of 8" in _error(ffn(None, 4, None, 2, 12, 8, 1, None, None, None, None, None, None))
    assert "experts" in _error(ffn(None, 4, None, 1025, 16, 8, 1, None, None, None, None, None, None))
    assert "activation" in _error(ffn(None, 4, None, 2, 16, 8, 2, None, None, None, None, None, None))
    assert "16-byte" in _error(ffn(8, 4, None, 2, 16, 8, 1, None, None, None, None, None, None))
    one, three = (ctypes.c_int64 * 1)(4), bytes([3])
    norm = f("zepp_op_grad_norm")
    assert "element type" in _error(norm((ctypes.c_void_p * 1)(16), one, three, 1, 1.0, 16, 16, None))
    assert "aligned" in _error(norm((ctypes.c_void_p * 1)(2), one, bytes([0]), 1, 1.0, 16, 16, None))
    # what a call cannot do without
    for rc in (f("zepp_op_gate")(None, 0, 1, 8, 2, 0, 1, None, 1.0, 16, 16, None),
               f("zepp_op_gate_grad")(16, 0, 1, 8, 2, 0, 1, 1.0, 16, 16, None, 16, None),
               f("zepp_op_sort")(16, 0, 1, 2, 8, None, None, 0, 8, None, 16, 16, 16, None),
               f("zepp_op_unsort")(16, 0, 1, 2, 8, None, None, 16, None),
               f("zepp_op_unsort_grad")(None, 16, 0, 1, 2, 8, 4, 16, 16, None, 16, None, None),
               ffn(16, 4, None, 2, 16, 8, 1, 16, 16, 16, None, 16, None),
               f("zepp_op_expert_ffn_grad")(16, 16, 4, 16, 2, 16, 8, 1, 16, 16, 16, 16, None, 16, None, None, None),
               norm((ctypes.c_void_p * 1)(0), one, bytes([0]), 1, 1.0, 16, 16, None), norm(None, None, None, 1, 1.0, 16, 16, None),
               norm(None, None, None, 0, 1.0, None, 16, None)):
        assert "null pointer" in _error(rc)


def test_sizes():
    assert ops._fn("zepp_op_sort_ws_ints")(1024, 8, 128) == 0                  # counted by every block itself
    assert ops._fn("zepp_op_sort_ws_ints")(1025, 8, 128) == 64 * 128
    assert ops._fn("zepp_op_grad_norm_ws_bytes")(1) >= 148 * 8 * 8


@pytest.mark.parametrize("tensor, dense", [
    (torch.zeros(4, 6), True), (torch.zeros(4, 6).t(), True), (torch.zeros(2, 4, 6).permute(1, 0, 2), True),
    (torch.zeros(4, 6)[:, :5], False), (torch.zeros(6).expand(4, 6), False), (torch.zeros(4, 1, 6).expand(4, 1, 6), True),
    (torch.zeros(8)[::2], False), (torch.zeros(1), True), (torch.zeros(()), True)])
def test_dense(tensor, dense):
    assert ops._is_dense(tensor) == dense
