"""The operators' edges that need no GPU: refusals, verdicts and sizes."""
import collections

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import zepp_b200 as zb
from zepp_b200 import ops
from zepp_b200._ext import lib


def error(rc):
    assert rc != 0
    return lib().zepp_last_error().decode()


def test_wait_limit():
    for ns in (-1, 3600 * 10 ** 9 + 1, 2 ** 62):
        assert "wait limit" in error(ops._fn("zepp_op_set_wait_limit_ns")(ns))
    for look in (zb.check_waits, ops.wait_failures):
        with pytest.raises(AssertionError, match="CUDA device"):
            look("cpu")
    for bad in (-1.0, float("nan"), float("inf"), 3601):
        with pytest.raises(AssertionError):
            ops.set_wait_limit(bad)
    ops.set_wait_limit(2)


class Device:
    """A device's status words: a failure is there until it is read, as zepp_op_status clears it."""

    def __init__(self):
        self.words = [0] * 8

    def fail(self, what):
        if not self.words[0]:
            self.words = [1, what, 2, 3, 0, 0, 0, 0]

    def read(self, index):
        words, self.words = self.words, [0] * 8
        return words


@pytest.fixture
def device(monkeypatch):
    d = Device()
    monkeypatch.setattr(ops, "_status", d.read)
    monkeypatch.setattr(ops, "_waits", {})
    return d


Config = collections.namedtuple("Config", "ranks swap shape", defaults=(None,))


def layer(device, status=(0,) * 8, trained=True):
    """As much of a layer as its verdict needs."""
    from zepp_b200.layer import EPMoE
    l = EPMoE.__new__(EPMoE)
    torch.nn.Module.__init__(l)
    l.w1 = l.w2 = None
    l.cfg = Config(ranks=1, swap=False)
    l.device, l._group_of, l._waits_seen, l.caps = torch.device("cuda", 0), torch.zeros(1) if trained else None, 0, None
    l._h = type("Handle", (), {"status": lambda self: list(status)})()
    return l


def test_a_failed_wait_is_told_to_everybody_once(device):
    a, b = layer(device), layer(device)
    for l in (a, b):
        l.check()
    zb.check_waits(0)
    device.fail(7)
    for look in (a.check, lambda: zb.check_waits(0), b.check):
        with pytest.raises(RuntimeError, match="wait id 7, item 2, step 3"):
            look()
        look()
    assert ops.wait_failures(0) == 1
    device.fail(8)
    device.fail(9)                                       # the first one of those not yet read is kept
    with pytest.raises(RuntimeError, match="wait id 8"):
        zb.check_waits("cuda:0")
    with pytest.raises(RuntimeError, match="wait id 8"):
        b.check()
    assert ops.wait_failures(0) == 2


def test_a_layers_own_failure_and_the_operators_are_both_told(device):
    device.fail(7)
    with pytest.raises(RuntimeError, match="step failed.*wait id 5.*operator failed.*wait id 7"):
        layer(device, status=(1, 5, 0, 0, 0, 0, 0, 0)).check()
    with pytest.raises(RuntimeError, match="step failed"):
        layer(device, status=(1, 5, 0, 0, 0, 0, 0, 0), trained=False).check()


@pytest.mark.parametrize("tokens, k", [(1 << 62, 4), ((1 << 61) + 1, 8), ((1 << 58) + 5, 64), (1 << 31, 1)])
def test_token_counts_whose_product_wraps_are_refused(tokens, k):
    for rc in (ops._fn("zepp_op_sort")(None, 0, tokens, k, 8, None, None, 0, 8, None, None, None, None, None),
               ops._fn("zepp_op_unsort")(None, 0, tokens, k, 8, None, None, None, None),
               ops._fn("zepp_op_unsort_grad")(None, None, 0, tokens, k, 8, 8, None, None, None, None, None, None)):
        assert "32-bit" in error(rc)


def test_clipping_refuses_parameters():
    """It scales what it is given: parameters instead of their gradients would be shrunk."""
    p = torch.nn.Parameter(torch.ones(3))
    for tensors in ([p], [torch.ones(3), p], (q for q in (p,))):
        with pytest.raises(AssertionError, match="leaf"):
            zb.clip_grad_norm_(tensors, 1.0)
    assert bool((p == 1).all())


def test_clipping_a_layer_without_gradients(device):
    l = layer(device)
    l.device = torch.device("cpu")
    for w, others in ((None, ()), (torch.zeros(2, requires_grad=True), [torch.zeros(3, requires_grad=True)])):
        l.w1 = l.w2 = w
        norm = l.clip_grad_norm_(1.0, others=others)
        assert norm.shape == () and norm.dtype == torch.float32 and float(norm) == 0.0


@pytest.mark.parametrize("ranks, swap", [(2, False), (1, True), (8, True)])
def test_training_calls_are_for_one_rank_without_swap(device, ranks, swap):
    l = layer(device)
    l.w1, l.w2 = torch.zeros(2), torch.zeros(2)
    l.cfg = Config(ranks, swap)
    for call in (l.train_weights, lambda: l.forward_train(None, None, None), lambda: l.clip_grad_norm_(1.0)):
        with pytest.raises(AssertionError, match="one rank, without swap"):
            call()
    assert not l.w1.requires_grad and not l.w2.requires_grad


def test_tensors_with_a_tangent():
    t = torch.ones(3)
    with fwAD.dual_level():
        d = fwAD.make_dual(t, t)
        ops._no_tangents(t, None, torch.zeros(2, dtype=torch.int32))
        for some in ((d,), (t, d), (None, d)):
            with pytest.raises(AssertionError, match="tangent"):
                ops._no_tangents(*some)
    ops._no_tangents(t, d)
