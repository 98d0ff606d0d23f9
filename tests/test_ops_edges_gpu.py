"""The operators around the layer at their edges: what neighbours, special values, streams and failures may not change."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import zepp_b200 as zb
from zepp_b200 import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def same_places(got, want):
    """NaN, +inf and -inf in the same places."""
    return (torch.equal(got.isnan(), want.isnan()) and torch.equal(got == math.inf, want == math.inf)
            and torch.equal(got == -math.inf, want == -math.inf))


# ------------------------------------------------------------------------------------------------------------- gate
@pytest.mark.parametrize("G, k", [(40, 4), (128, 8), (384, 8), (1000, 32)])
@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gate_gradient_of_rows_with_nan(G, k, score, renormalize, dtype):
    """A row's NaN makes its weights NaN and with them the gradients of the experts that it chose, or of all experts where
    the weights are probabilities over all of them; it reaches no other row.  What is masked with -inf besides stays out."""
    g = gen(G + k)
    clean, dw = randn((12, G), g, dtype, 2.0), randn((12, k), g)
    l = clean.clone()
    l[1, 5] = math.nan                                # one
    l[4] = math.nan                                   # nothing else
    l[7, 2], l[7, 3:] = math.nan, -math.inf           # two experts left to choose
    res = []
    for t in (clean, l):
        t = t.clone().requires_grad_(True)
        ids, w = zb.route_topk(t, k, score=score, renormalize=renormalize)
        res.append((ids, w.detach(), torch.autograd.grad(w, t, dw)[0]))
    (_, w0, d0), (ids, w, d) = res
    bad = torch.tensor([1, 4, 7], device="cuda")
    good = torch.tensor([i for i in range(12) if i not in (1, 4, 7)], device="cuda")
    assert torch.equal(w[good], w0[good]) and torch.equal(d[good], d0[good]) and bool(w[bad].isnan().all())
    assert bool((ids[1] != 5).all()) and bool((ids[4] == -1).all()) and sorted(ids[7].tolist())[-2:] == [0, 1] and bool((ids[7, 2:] == -1).all())
    want = torch.zeros((12, G), device="cuda")
    if score == "softmax" and not renormalize:
        want[bad] = math.nan
    else:
        want[1, ids[1].long()] = math.nan
        want[7, :2] = math.nan
    assert same_places(d[bad].float(), want[bad]) and bool((d[bad].nan_to_num(0.0) == 0).all())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gate_of_rows_with_an_infinite_logit(score):
    """+inf is chosen first.  Its sigmoid is 1 with slope 0; its softmax is inf - inf."""
    l = randn((3, 20), gen(1))
    l[1, 6] = math.inf
    l.requires_grad_(True)
    ids, w = zb.route_topk(l, 3, score=score, renormalize=False)
    d = torch.autograd.grad(w, l, torch.ones_like(w))[0]
    assert int(ids[1, 0]) == 6 and bool(w[::2].isfinite().all()) and bool(d[::2].isfinite().all())
    if score == "sigmoid":
        assert float(w.detach()[1, 0]) == 1.0 and float(d[1, 6]) == 0.0 and bool(d[1].isfinite().all())
    else:
        assert bool(w[1, 0].isnan()) and bool(d[1, 6].isnan())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_infinities_keep_their_sign(dtype):
    """Rows, sums and gradients that are infinite: the same sign as by the formulas."""
    g = gen(5)
    T, K, H = 30, 4, 64
    ids = torch.randint(0, 6, (T, K), generator=g, device="cuda", dtype=torch.int32)
    x = randn((T, H), g, dtype)
    x[3, 5], x[4, 6], x[8] = math.inf, -math.inf, -math.inf
    rows, plan = zb.sort_tokens(x, ids, 6)
    at = plan.position.long()
    assert torch.equal(rows[at], x[:, None, :].expand(T, K, H))
    w = randn((T, K), g)
    w[8] = torch.tensor([1.0, 2.0, 0.5, 3.0], device="cuda")
    r, w = rows.clone().requires_grad_(True), w.requires_grad_(True)
    y = zb.unsort_tokens(r, plan, w)
    want = (rows.double()[at] * w.detach().double()[..., None]).sum(1)
    assert same_places(y.detach().double(), want) and bool((y[8] == -math.inf).all())
    dy = randn((T, H), g, dtype)
    dy[2], dy[11, 7] = math.inf, -math.inf
    dr, dw = torch.autograd.grad(y, (r, w), dy)
    assert same_places(dr[at].double(), w.detach().double()[..., None] * dy.double()[:, None, :])
    assert same_places(dw.double(), (rows.double()[at] * dy.double()[:, None, :]).sum(2))
    grads = [x.clone()]
    assert math.isinf(float(zb.grad_norm(grads))) and float(zb.grad_norm([-x[:3].float(), torch.full((1,), -math.inf, device="cuda")])) == math.inf


U = 2.0 ** -24


@pytest.mark.parametrize("T, K, H, dtype", [(650, 11, 2056, torch.float16), (592, 1, 2048, torch.bfloat16), (593, 9, 6152, torch.bfloat16), (1200, 24, 2048, torch.float16),
                                            (591, 8, 4096, torch.bfloat16), (700, 8, 1024, torch.bfloat16), (700, 3, 4096, torch.float32)])
def test_unsort_gradient_of_long_rows(T, K, H, dtype):
    """Both ways that the gradient of long rows is computed: whole pieces and ragged ones, one copy and more than eight, tokens
    without any, the two results together and each alone."""
    g = gen(T + K)
    ids = torch.randint(-1, 40, (T, K), generator=g, device="cuda", dtype=torch.int32)
    ids[7], ids[T - 1] = -1, -1
    _, plan = zb.sort_tokens(randn((T, 8), g), ids, 40)
    r, w, dy = randn((T * K, H), g, dtype).requires_grad_(True), randn((T, K), g).requires_grad_(True), randn((T, H), g, dtype)
    dr, dw = torch.autograd.grad(zb.unsort_tokens(r, plan, w), (r, w), dy)
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny
    dr64 = torch.zeros((T * K, H), dtype=torch.float64, device="cuda")
    for k in range(K):
        p = plan.position[:, k].long()
        t = (p >= 0).nonzero()[:, 0]
        dr64[p[t]] = w.detach()[t, k, None].double() * dy[t].double()
        d = r.detach()[p.clamp_min(0)].double() * dy.double() * (p >= 0)[:, None]
        # a thread adds at most H / 32 products one after the other, then 5 + 8 sums join them
        bound = (H / 32 + 8 + 13) * U * d.abs().sum(1) + 1e-30
        assert bool(((dw[:, k].double() - d.sum(1)).abs() <= bound).all()) and bool((dw[p < 0, k] == 0).all())
    assert bool(((dr.double() - dr64).abs() <= (half + 2 * U) * dr64.abs() + tiny).all())
    assert torch.equal(torch.autograd.grad(zb.unsort_tokens(r, plan, w.detach()), r, dy)[0], dr)
    assert torch.equal(torch.autograd.grad(zb.unsort_tokens(r.detach(), plan, w), w, dy)[0], dw)
    ops.check_waits()


# -------------------------------------------------------------------------------------------------- experts' products
@pytest.mark.parametrize("act, experts, most, H, I", [("swiglu", 200, 150, 512, 256), ("gelu", 97, 400, 1032, 264), ("swiglu", 600, 31, 256, 128)])
def test_expert_ffn_rows_of_neighbours_never_reach_a_weight_gradient(act, experts, most, H, I):
    """The last step of an expert's sum holds rows of the next expert, which are cleared by both CTAs of a pair.  Over many
    waves of tiles, with NaN and infinities in every second expert's rows, the experts between them get the same bits as
    with clean neighbours, every time."""
    g = gen(experts)
    counts = torch.randint(0, most, (experts,), generator=g, device="cuda")
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    n = int(offsets[-1])
    f1 = I * (2 if act == "swiglu" else 1)
    x, dy = randn((n, H), g, torch.bfloat16), randn((n, H), g, torch.bfloat16)
    w1, w2 = randn((experts, f1, H), g, torch.bfloat16, H ** -0.5), randn((experts, H, I), g, torch.bfloat16, I ** -0.5)
    expert = torch.repeat_interleave(torch.arange(experts, device="cuda"), counts)
    odd = (expert % 2 == 1)[:, None]
    res = []
    for change in (lambda t, v: t, lambda t, v: torch.where(odd, torch.full_like(t, v), t)):
        leaves = [change(x, math.nan).requires_grad_(True), w1.clone().requires_grad_(True), w2.clone().requires_grad_(True)]
        y = zb.expert_ffn(leaves[0], offsets, leaves[1], leaves[2], act=act)
        for _ in range(20 if res else 1):
            _, d1, d2 = torch.autograd.grad(y, leaves, change(dy, math.inf), retain_graph=True)
            res.append((d1[::2], d2[::2]))
    assert bool(res[0][0].isfinite().all()) and bool(res[0][1].isfinite().all())
    for a, b in res[1:]:
        assert torch.equal(a, res[0][0]) and torch.equal(b, res[0][1])
    ops.check_waits()


# ------------------------------------------------------------------------------------------------ sort by expert and back
def test_sort_with_an_empty_group_table():
    """No id has a group in it, so no copy gets a row."""
    x = randn((5, 16), gen(1)).requires_grad_(True)
    ids = torch.arange(10, dtype=torch.int32, device="cuda").view(5, 2) % 4
    rows, plan = zb.sort_tokens(x, ids, 4, group_of=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert not plan.offsets.any() and bool((plan.position == -1).all()) and not rows.any()
    assert not torch.autograd.grad(rows, x, torch.ones_like(rows))[0].any()


# ------------------------------------------------------------------------------------------------------- refusals
def test_sizes_beyond_the_limits_are_refused():
    """Before anything is allocated or launched, with the error that the other arguments have."""
    one = torch.zeros((), dtype=torch.bfloat16, device="cuda")
    zero = torch.zeros((), dtype=torch.int32, device="cuda")
    H = (1 << 20) + 8
    plan = ops.SortPlan(zero.expand(5), zero.expand(1, 2))
    many = ops.SortPlan(zero.expand(5), zero.expand(1 << 30, 2))
    for call in (
            lambda: zb.sort_tokens(one.expand(1, H), zero.expand(1, 2), 4),
            lambda: zb.sort_tokens(one.expand(1 << 30, 8), zero.expand(1 << 30, 2), 4),
            lambda: zb.unsort_tokens(one.expand(2, H), plan),
            lambda: zb.unsort_tokens(one.expand(1 << 31, 8), many),
            lambda: zb.expert_ffn(one.expand(2, H), zero.expand(2), one.expand(1, 16, H), one.expand(1, H, 8)),
            lambda: zb.expert_ffn(one.expand(2, 8), zero.expand(2), one.expand(1, H, 8), one.expand(1, 8, H), act="gelu"),
            lambda: zb.expert_ffn(one.expand(1 << 31, 8), zero.expand(2), one.expand(1, 16, 8), one.expand(1, 8, 8))):
        with pytest.raises(AssertionError, match="2\\^31|up to|at most"):
            call()


# ------------------------------------------------------------------------------------------------- waits that run out
@pytest.fixture
def no_patience():
    ops.set_wait_limit(0)
    yield
    ops.set_wait_limit(2)
    torch.cuda.synchronize()


def long_sums(n):
    """One expert with so many rows that a weight gradient's accumulators take long: the epilogue has to wait for them."""
    rows = torch.ones((n, 8), dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    w1 = torch.full((1, 8, 8), 0.125, dtype=torch.bfloat16, device="cuda")
    w2 = torch.zeros((1, 8, 8), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    return zb.expert_ffn(rows, offsets, w1, w2, act="gelu"), w2, rows


def test_a_wait_that_runs_out_is_reported_and_leaves_the_gpu_usable(no_patience):
    """Without patience the epilogue gives up at once, with the copies and products of both CTAs in flight: the kernel ends
    by itself, the verdict names it, and the next call is right."""
    ops.set_wait_limit(2)
    y, w2, dy = long_sums(1 << 26)
    want = torch.autograd.grad(y, w2, dy, retain_graph=True)[0]
    torch.cuda.synchronize()
    ops.check_waits()
    for _ in range(3):
        ops.set_wait_limit(0)
        torch.autograd.grad(y, w2, dy, retain_graph=True)
        torch.cuda.synchronize()
        ops.set_wait_limit(2)
        with pytest.raises(RuntimeError, match="wait ran out"):
            ops.check_waits()
        assert torch.equal(torch.autograd.grad(y, w2, dy, retain_graph=True)[0], want)
        torch.cuda.synchronize()
        ops.check_waits()


def test_a_wait_that_runs_out_on_another_stream_is_reported(no_patience):
    """The backward pass runs on its forward pass's stream, which is still busy when another one asks."""
    ops.set_wait_limit(2)
    ops.check_waits()
    before = ops.wait_failures()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y, w2, dy = long_sums(1 << 26)
        torch.cuda._sleep(200_000_000)                   # about a tenth of a second before the kernel starts
        ops.set_wait_limit(0)
        torch.autograd.grad(y, w2, dy)
        ops.set_wait_limit(2)
    with pytest.raises(RuntimeError, match="wait ran out"):
        ops.check_waits(torch.device("cuda"))
    assert ops.wait_failures("cuda:0") == before + 1
    ops.check_waits()


@pytest.mark.parametrize("spare", (0, 3))
def test_a_long_sum_is_waited_for(no_patience, spare):
    """The epilogue's wait for a sum over all rows of an expert grows with their number: it does not run out because there
    are many.  2^26 rows are 2^20 steps, for which the limit is twice what was set.  With three rows more the last
    step holds rows behind the expert's, whose clearing waits as long."""
    ops.set_wait_limit(2)
    y, w2, dy = long_sums((1 << 26) + spare)
    torch.autograd.grad(y, w2, dy, retain_graph=True)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    want = torch.autograd.grad(y, w2, dy, retain_graph=True)[0]
    end.record()
    torch.cuda.synchronize()
    ops.check_waits()
    ops.set_wait_limit(0.7 * start.elapsed_time(end) / 1e3)
    got = torch.autograd.grad(y, w2, dy)[0]
    ops.check_waits()
    assert torch.equal(got, want)


# --------------------------------------------------------------------------------------------- norm of many, clipping
def test_clipping_takes_gradients_and_no_parameters():
    p = torch.nn.Parameter(torch.full((50,), 2.0, device="cuda"))
    with pytest.raises(AssertionError, match="leaf"):
        zb.clip_grad_norm_([p], 1.0)
    assert bool((p == 2).all())
    grads = torch.autograd.grad(p.square().sum(), p, create_graph=True)       # of a graph, but not a leaf
    zb.clip_grad_norm_(grads, 1.0)
    # 50 squares of 4: norm 4 sqrt(50); the factor, the product and the root round once each
    assert bool(((grads[0].detach().double() * 50 ** 0.5 - 1).abs() <= 4 * 2.0 ** -24 + 1e-6).all())
    assert float(zb.grad_norm([p])) > 0                                       # only reads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size, max_norm", [(1e38, 1.0), (1e38, 1e-3), (3e38, 1e-6), (1e38, 1e-9), (3e38, 30.0)])
def test_clipping_by_factors_below_the_normal_numbers(dtype, size, max_norm):
    """Elements near the top of the range: the factor has fewer bits than fp32's normal numbers, the result has all."""
    t = (torch.rand(1000, generator=gen(7), device="cuda") * size).to(dtype)
    want = t.double()
    total = float(want.norm())
    want = want * min(1.0, max_norm / (total + 1e-6))
    zb.clip_grad_norm_([t], max_norm)
    # sums of at most 64 squares in fp32 (half of it in the root), the quotient, the product and the result's own rounding
    bound = (torch.finfo(dtype).eps / 2 + 40 * 2.0 ** -24) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((t.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("special", [1.0, math.inf, -math.inf, math.nan])
def test_clipping_with_an_infinite_limit(special):
    """No limit: nothing changes, whatever the norm, but for a norm of NaN."""
    t = randn((500,), gen(3))
    t[17] = special
    kept = t.clone()
    norm = zb.clip_grad_norm_([t], math.inf)
    if math.isnan(special):
        assert math.isnan(float(norm)) and bool(t.isnan().all())
    else:
        assert torch.equal(t, kept) and math.isinf(float(norm)) == math.isinf(special)


# ------------------------------------------------------------------------------------------------- forward-mode derivatives
def test_inputs_with_a_tangent_are_refused():
    """A dual tensor does not require a gradient; its tangent would be dropped, which is a derivative of zero."""
    i32, bf = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.bfloat16, device="cuda")
    l, x, w = (torch.rand(*s, device="cuda") for s in ((4, 8), (4, 16), (4, 2)))
    ids = torch.arange(8, **i32).view(4, 2)
    rows, plan = zb.sort_tokens(x, ids, 8)
    a, w1, w2, off = torch.rand(4, 16, **bf), torch.rand(2, 16, 16, **bf), torch.rand(2, 16, 8, **bf), torch.tensor([0, 1, 4], **i32)
    calls = [(lambda l: zb.route_topk(l, 2), (l,)), (lambda x: zb.sort_tokens(x, ids, 8), (x,)),
             (lambda r, w: zb.unsort_tokens(r, plan, w), (rows, w)), (lambda a, u, v: zb.expert_ffn(a, off, u, v), (a, w1, w2)),
             (lambda t: zb.grad_norm([l, t]), (x,)), (lambda t: zb.clip_grad_norm_([l, t], 1.0), (x,))]
    for call, args in calls:
        kept = [t.clone() for t in args]
        with fwAD.dual_level():
            for i in range(len(args)):
                with pytest.raises(AssertionError, match="tangent"):
                    call(*[fwAD.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)])
            call(*args)                                                           # without a tangent
        if call is not calls[-1][0]:
            assert all(torch.equal(t, k) for t, k in zip(args, kept))
    with fwAD.dual_level(), pytest.raises((AssertionError, RuntimeError)):        # as well as a gradient: still no silent zero
        zb.unsort_tokens(fwAD.make_dual(rows, torch.ones_like(rows)), plan, w.requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: zb.route_topk(t, 2)[1])(l[None].expand(3, 4, 8))
    with pytest.raises((AssertionError, RuntimeError)):
        torch.func.jvp(lambda t: zb.route_topk(t, 2)[1], (l,), (torch.ones_like(l),))
