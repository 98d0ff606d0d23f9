"""The operators around the layer against plain implementations in 64 bits.

Tolerances count roundings: half a step of a type is `finfo(t).eps / 2` relative to the value, U = 2^-24 that of fp32."""
import dataclasses
import math

import pytest
import torch

import zepp_b200 as zb
from zepp_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere, NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    far = ((got - want).abs() - bound).nan_to_num(0.0, 0.0, 0.0)
    assert torch.equal(got.isinf(), want.isinf()), what
    assert bool((far <= 0).all()), (what, float(far.max()), int(far.argmax()))


# ------------------------------------------------------------------------------------------------------------- gate
def gate64(l, k, score, renormalize, bias, scale):
    """ids and differentiable weights in 64 bits, one place after the other."""
    T, G = l.shape
    d = l.detach().double()
    key = d.clone()
    if bias is not None:
        key = torch.sigmoid(d) + bias.double()
        key[d == -math.inf] = -math.inf
    key[d.isnan()] = -math.inf
    key = torch.where(key.isnan(), torch.full_like(key, -math.inf), key)
    ids = torch.full((T, k), -1, dtype=torch.int64, device=l.device)
    for j in range(k):
        top = key.max(1, keepdim=True).values
        at = (key == top).to(torch.int8).argmax(1)               # the first one
        ok = top[:, 0] > -math.inf
        ids[ok, j] = at[ok]
        key.scatter_(1, at[:, None], -math.inf)
    z = l.double()
    there = ids >= 0
    zc = z.gather(1, ids.clamp_min(0))
    if score == "sigmoid":
        v = torch.where(there, torch.sigmoid(zc), torch.zeros_like(zc))
        w = v / (v.sum(1, keepdim=True) + 1e-20) if renormalize else v
    else:
        low = torch.full_like(z, -1e300)
        safe = torch.where(z == -math.inf, low, z)
        e = torch.exp(safe - torch.where(z.isnan(), low, safe).detach().amax(1, keepdim=True))
        e = torch.where(z == -math.inf, torch.zeros_like(e), e)
        v = torch.where(there, e.gather(1, ids.clamp_min(0)), torch.zeros_like(zc))
        total = v.sum(1, keepdim=True) if renormalize else e.sum(1, keepdim=True)
        w = v / torch.where(total == 0, torch.ones_like(total), total)
    w = w * scale
    return ids.int(), torch.where(d.isnan().any(1, keepdim=True), torch.full_like(w, math.nan), w)


def gate_case(T, G, k, score, renormalize, with_bias, dtype, seed, std=2.0, scale=1.0, change=None):
    g = gen(seed)
    l = randn((T, G), g, dtype, std)
    if change is not None:
        change(l)
    bias = randn((G,), g, std=0.1) if with_bias else None
    dw = randn((T, k), g)
    l.requires_grad_(True)
    ids, w = zb.route_topk(l, k, score=score, renormalize=renormalize, bias=bias, scale=scale)
    m = l.detach().double().requires_grad_(True)
    ids64, w64 = gate64(m, k, score, renormalize, bias, scale)
    assert ids.dtype == torch.int32 and torch.equal(ids, ids64)
    # exp of a difference of logits: the difference is rounded once (relative to its size), expf is off by 2 units, the
    # sum by its depth (NPL + 5), quotient and scale by one each
    fin = l.detach().double()
    fin = torch.where(fin.isfinite(), fin, torch.zeros_like(fin))
    spread = float((fin.amax(1) - fin.amin(1)).max()) if T else 0.0
    rel = (spread + 2 * 2 * 2 + 40 + 4) * U
    within(w.detach(), w64.detach(), rel * w64.detach().abs() + 1e-30, "weights")
    if not T:
        assert torch.autograd.grad(w, l, dw)[0].shape == (0, G)
        return
    dl = torch.autograd.grad(w, l, dw)[0]
    dl64 = torch.autograd.grad(w64, m, torch.where(ids64 >= 0, dw.double(), torch.zeros_like(dw.double())))[0]
    # dl_c = v_c (q_c - sum q v): both terms carry the weights' relative error, in sum at most twice the row's largest product
    size = scale * dw.double().abs().amax(1, keepdim=True) * 2
    within(dl, dl64.nan_to_num(0.0) if change is None else dl64, HALF[dtype] * dl64.abs() + 3 * rel * size + torch.finfo(dtype).tiny, "dlogits")


@pytest.mark.parametrize("T, G, k", [(1, 8, 2), (0, 8, 2), (3, 1, 1), (37, 129, 8), (64, 384, 8), (5, 33, 32), (130, 128, 8), (9, 1000, 10), (17, 1024, 32), (40, 500, 6)])
@pytest.mark.parametrize("score, renormalize, with_bias", [("softmax", True, False), ("softmax", False, False), ("sigmoid", True, True), ("sigmoid", False, False), ("sigmoid", False, True)])
def test_gate(T, G, k, score, renormalize, with_bias):
    for i, dtype in enumerate(TYPES):
        gate_case(T, G, k, score, renormalize, with_bias, dtype, 100 + i, scale=(1.0, 2.5, 0.5)[i])


@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gate_masked_rows_and_ties(score, renormalize):
    def mask(l):
        l[0] = -math.inf                       # a pad row
        l[1, 2:] = -math.inf                   # fewer experts than k
        l[2] = 1.0                             # all equal: the lowest indices
        l[3] = torch.finfo(l.dtype).min        # the type's lowest value is a value
        l[4, ::2] = 0.0
        l[4, 1::2] = -0.0                      # equal
        l[5, 7] = -math.inf
    gate_case(8, 64, 6, score, renormalize, False, torch.float32, 7, change=mask)
    gate_case(8, 64, 6, score, renormalize, False, torch.bfloat16, 8, change=mask)


def test_gate_ids_of_rows_with_nan_and_inf():
    l = torch.randn(4, 40, generator=gen(3), device="cuda")
    l[0, 5] = math.nan
    l[1, 6] = math.inf
    l[2] = math.nan
    for score in ("softmax", "sigmoid"):
        ids, w = zb.route_topk(l, 4, score=score)
        assert 5 not in ids[0].tolist() and bool(w[0].isnan().all()) and ids[1, 0] == 6
        assert ids[2].tolist() == [-1] * 4 and bool(w[2].isnan().all())
        assert bool(w[3].isfinite().all()) and bool(((ids[3] >= 0) & (ids[3] < 40)).all())


def test_gate_choice_by_bias_is_exact_between_near_equals():
    """Scores that agree in fp32: the choice is that of 64 bits, equal ones by index."""
    G = 96
    l = torch.full((64, G), 12.0, device="cuda")
    l += torch.arange(G, device="cuda")[None, :] * 1e-4 * torch.randint(-3, 4, (64, 1), generator=gen(1), device="cuda")
    bias = torch.zeros(G, device="cuda")
    for b in (bias, bias + 0.25):
        ids, _ = zb.route_topk(l, 8, score="sigmoid", bias=b)
        want, _ = gate64(l, 8, "sigmoid", True, b, 1.0)
        assert torch.equal(ids, want)


def test_gate_strides_and_alignment():
    g = gen(5)
    base = randn((33, 264), g)
    for l in (base[:, 3:131], base[:, 1:257:2], randn((130, 33), g).t(), randn((33 * 128 + 1,), g)[1:].view(33, 128)):
        a, wa = zb.route_topk(l, 8)
        b, wb = zb.route_topk(l.clone().contiguous(), 8)
        assert torch.equal(a, b) and torch.equal(wa, wb)


# ------------------------------------------------------------------------------------------------ sort by expert and back
def sort64(x, ids, G):
    T, K = ids.shape
    flat = ids.reshape(-1).tolist()
    order = sorted((i for i, e in enumerate(flat) if 0 <= e < G), key=lambda i: (flat[i], i))
    position = torch.full((T * K,), -1, dtype=torch.int32)
    for row, i in enumerate(order):
        position[i] = row
    offsets = torch.tensor([sum(1 for e in flat if 0 <= e < g) for g in range(G + 1)], dtype=torch.int32)
    rows = torch.zeros((T * K, x.shape[1]), dtype=x.dtype, device=x.device)
    if order:
        rows[:len(order)] = x[torch.tensor(order, device=x.device) // K]
    return rows, offsets.to(x.device), position.view(T, K).to(x.device)


@pytest.mark.parametrize("T, K, G, H", [(1, 1, 1, 1), (1, 8, 128, 2048), (0, 4, 8, 64), (7, 3, 5, 1003), (64, 8, 128, 136), (300, 64, 17, 24),
                                        (1100, 8, 384, 40), (2050, 5, 2048, 17), (513, 6, 3, 256)])
def test_sort_and_back(T, K, G, H):
    for i, dtype in enumerate(TYPES):
        g = gen(T + K + G + H + i)
        ids = torch.randint(-1, G, (T, K), generator=g, device="cuda", dtype=torch.int32)     # pads, and experts taken twice
        if T:
            ids[0, 0] = G + 3                                                                 # not an expert: no row
        x = randn((T, H), g, dtype).requires_grad_(True)
        rows, plan = zb.sort_tokens(x, ids, G)
        want = sort64(x.detach(), ids, G)
        assert torch.equal(rows, want[0]) and torch.equal(plan.offsets, want[1]) and torch.equal(plan.position, want[2])
        r = randn((T * K, H), g, dtype).requires_grad_(True)
        w = randn((T, K), g).requires_grad_(True)
        y = zb.unsort_tokens(r, plan, w)
        took = (plan.position >= 0).double()
        pick = r.detach().double()[plan.position.clamp_min(0).long()] if T else torch.zeros(T, K, H, device="cuda", dtype=torch.float64)
        pick = pick * took[..., None]
        wd = w.detach().double()
        size = (pick.abs() * wd.abs()[..., None]).sum(1)
        y64 = (pick * wd[..., None]).sum(1)
        within(y, y64, HALF[dtype] * y64.abs() + 2 * K * U * size + torch.finfo(dtype).tiny, "y")
        dy = randn((T, H), g, dtype)
        dr, dw = torch.autograd.grad(y, (r, w), dy)
        dr64 = torch.zeros((T * K, H), dtype=torch.float64, device="cuda")
        t, k = (plan.position >= 0).nonzero(as_tuple=True)
        dr64[plan.position[t, k].long()] = wd[t, k, None] * dy.double()[t]
        within(dr, dr64, (HALF[dtype] + 2 * U) * dr64.abs() + torch.finfo(dtype).tiny, "drows")
        d = dy.double()[:, None, :] * pick
        # a thread adds at most H / 32 products one after the other, then 5 + 8 sums join them
        within(dw, d.sum(2), (H / 32 + 8 + 13) * U * d.abs().sum(2) + 1e-30, "dweights")
        ds = randn((T * K, H), g, dtype)
        dx = torch.autograd.grad(rows, x, ds)[0]
        back = (ds.double()[plan.position.clamp_min(0).long()] if T else torch.zeros(T, K, H, device="cuda", dtype=torch.float64)) * took[..., None]
        within(dx, back.sum(1), HALF[dtype] * back.sum(1).abs() + K * U * back.abs().sum(1) + torch.finfo(dtype).tiny, "dx")


def test_sort_keeps_nothing_of_rows_without_a_copy():
    """Rows behind the last copy are zero in the rows and in their gradient, whatever the memory held."""
    g = gen(9)
    x = randn((12, 64), g, torch.bfloat16)
    ids = torch.full((12, 4), -1, dtype=torch.int32, device="cuda")
    ids[3, 2], ids[5, 0] = 1, 0
    junk = torch.full((48, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    del junk
    rows, plan = zb.sort_tokens(x, ids, 2)
    assert plan.offsets.tolist() == [0, 1, 2] and bool((rows[2:] == 0).all())
    r = torch.full((48, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    r[:2] = rows[:2]
    r.requires_grad_(True)
    w = torch.full((12, 4), math.nan, device="cuda")          # of copies that have no row
    w[3, 2], w[5, 0] = 0.5, 2.0
    w.requires_grad_(True)
    y = zb.unsort_tokens(r, plan, w)
    assert bool(y.isfinite().all()) and torch.equal(y[5], 2 * x[5]) and bool((y[0] == 0).all())
    dr, dw = torch.autograd.grad(y.sum(), (r, w))             # an expanded gradient
    assert bool((dr[2:] == 0).all()) and bool((dr[0] == 2).all()) and bool((dw[plan.position < 0] == 0).all())


def test_sort_group_table_and_strides():
    g = gen(11)
    x = randn((50, 96), g, torch.bfloat16)
    ids = torch.randint(-1, 6, (50, 4), generator=g, device="cuda", dtype=torch.int32)
    table = torch.tensor([3, 1, 7, -1, 2, 9], dtype=torch.int32, device="cuda")        # 9 and -1: no group
    rows, plan = zb.sort_tokens(x, ids, 8, group_of=table)
    mapped = torch.where(ids >= 0, table[ids.clamp_min(0).long()], ids)
    want = sort64(x, mapped, 8)
    assert torch.equal(rows, want[0]) and torch.equal(plan.offsets, want[1]) and torch.equal(plan.position, want[2])
    wide = randn((50, 200), g, torch.bfloat16)
    for v in (wide[:, 1:97], wide[:, ::2][:, :96], randn((96, 50), g, torch.bfloat16).t(), randn((50 * 96 + 1,), g, torch.bfloat16)[1:].view(50, 96)):
        assert torch.equal(zb.sort_tokens(v, ids, 8)[0], zb.sort_tokens(v.clone().contiguous(), ids, 8)[0])
    shifted = randn((200 * 96 + 1,), g, torch.bfloat16)[1:].view(200, 96)              # rows off the 16-byte boundary
    assert torch.equal(zb.unsort_tokens(shifted, plan), zb.unsort_tokens(shifted.clone(), plan))


# -------------------------------------------------------------------------------------------------- experts' products
def act64(h, act, I):
    if act == "swiglu":
        return torch.nn.functional.silu(h[..., :I]) * h[..., I:]
    return torch.nn.functional.gelu(h)


def ffn64(x, off, w1, w2, act):
    I = w2.shape[2]
    out = [torch.zeros((0, x.shape[1]), dtype=torch.float64, device=x.device)]
    for e in range(w1.shape[0]):
        out.append(act64(x[off[e]:off[e + 1]] @ w1[e].T, act, I) @ w2[e].T)
    tail = x.shape[0] - off[-1]
    return torch.cat(out + [torch.zeros((tail, x.shape[1]), dtype=torch.float64, device=x.device)])


def ffn_inputs(counts, H, I, act, spare, seed):
    g = gen(seed)
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    n, G = off[-1] + spare, len(counts)
    f1 = I * (2 if act == "swiglu" else 1)
    x = randn((n, H), g, torch.bfloat16)
    if spare:
        x[off[-1]:] = math.nan                                 # behind the last expert: anything
    return (x, torch.tensor(off, dtype=torch.int32, device="cuda"), randn((G, f1, H), g, torch.bfloat16, H ** -0.5),
            randn((G, H, I), g, torch.bfloat16, I ** -0.5), randn((n, H), g, torch.bfloat16), off)


def near(got, want, what):
    """Outputs of products of operands that were rounded to bf16 once or twice on the way: the errors of the summands are
    independent, so the result is off by about sqrt(3) half-steps of its own root mean square (4 standard deviations of
    the rounding, one half-step / sqrt(3), per factor); 2^-7 of the norm leaves no room for a missing or doubled part."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape and bool(got.isfinite().all()), what
    if want.numel() == 0:
        return
    norm = float(want.norm())
    assert float((got - want).norm()) <= 2.0 ** -7 * norm + 1e-30, (what, float((got - want).norm()), norm)
    # and no single element further off than 2^-5 of the largest
    assert float((got - want).abs().max()) <= 2.0 ** -5 * float(want.abs().max()) + 1e-30, what


FFN_CASES = [
    ((1,), 8, 8, "swiglu", 0), ((0, 3, 0), 64, 64, "swiglu", 2), ((130, 0, 1, 64, 65, 127), 136, 72, "swiglu", 3),
    ((33, 16, 15, 17, 0, 48), 392, 136, "gelu", 5), ((300,), 256, 384, "swiglu", 0), ((129, 256, 40), 520, 264, "gelu", 0),
    ((0, 0), 128, 128, "swiglu", 4), (tuple(range(40)), 192, 128, "swiglu", 1), ((5,) * 128, 256, 128, "gelu", 0),
    ((500, 40, 0, 390), 520, 264, "swiglu", 0), ((3,) * 400, 136, 72, "swiglu", 1), ((2,) * 1024, 64, 64, "gelu", 0),
    # several column tiles of a weight gradient in a row, for experts short and long
    ((0, 1, 15, 16, 17, 63, 64, 65, 0, 383, 384, 385, 700) + tuple((7 * i) % 97 for i in range(115)), 1024, 512, "swiglu", 9)]


@pytest.mark.parametrize("counts, H, I, act, spare", FFN_CASES)
def test_expert_ffn(counts, H, I, act, spare):
    x, offsets, w1, w2, dy, off = ffn_inputs(counts, H, I, act, spare, sum(counts) + H)
    y0 = zb.expert_ffn(x, offsets, w1, w2, act=act)            # no gradient wanted
    leaves = [t.requires_grad_(True) for t in (x, w1, w2)]
    y = zb.expert_ffn(x, offsets, w1, w2, act=act)
    assert torch.equal(y, y0)
    dx, d1, d2 = torch.autograd.grad(y, leaves, dy)
    m = [t.detach().double().requires_grad_(True) for t in leaves]
    y64 = ffn64(m[0], off, m[1], m[2], act)
    end = off[-1]
    near(y[:end], y64[:end], "y")
    assert bool((y[end:] == 0).all())
    g64 = torch.autograd.grad(y64, m, dy.double())
    near(dx[:end], g64[0][:end], "dx")
    assert bool((dx[end:] == 0).all())
    near(d1, g64[1], "dw1")
    near(d2, g64[2], "dw2")
    for e, c in enumerate(counts):                             # per expert: a small one is not hidden by the others
        if c:
            near(d1[e], g64[1][e], ("dw1", e))
            near(d2[e], g64[2][e], ("dw2", e))
        else:
            assert bool((d1[e] == 0).all()) and bool((d2[e] == 0).all()), e
    ops.check_waits()


def test_expert_ffn_products_are_exact_where_they_can_be():
    """Small whole numbers: every product and sum is exact in fp32, and outputs below 256 in bf16; catches any operand
    element in a wrong place.  GELU is the identity up to rounding for large arguments and 0 for large negative ones."""
    g = gen(4)
    H, I, counts = 136, 72, (70, 0, 129, 3)
    n, G = sum(counts), len(counts)
    offsets = torch.tensor([0, 70, 70, 199, 202], dtype=torch.int32, device="cuda")
    x = torch.zeros((n, H), device="cuda")
    x.scatter_(1, torch.randint(0, H, (n, 1), generator=g, device="cuda"), 1.0)               # one-hot rows
    w1 = torch.randint(0, 2, (G, I, H), generator=g, device="cuda").float() * 128 - 64        # h = 64 or -64
    w2 = torch.zeros((G, H, I), device="cuda")
    w2.scatter_(2, torch.randint(0, I, (G, H, 1), generator=g, device="cuda"), 1.0)
    b = [t.bfloat16().requires_grad_(True) for t in (x, w1, w2)]
    y = zb.expert_ffn(b[0], offsets, b[1], b[2], act="gelu")
    dy = torch.zeros((n, H), device="cuda")
    dy.scatter_(1, torch.randint(0, H, (n, 1), generator=g, device="cuda"), 1.0)
    dx, d1, d2 = torch.autograd.grad(y, b, dy.bfloat16())
    off = offsets.tolist()
    for e in range(G):
        s = slice(off[e], off[e + 1])
        h = x[s] @ w1[e].T
        a = h.clamp_min(0)
        da = dy[s] @ w2[e]
        dh = da * (h > 0)
        assert torch.equal(y[s].float(), a @ w2[e].T), e
        assert torch.equal(dx[s].float(), dh @ w1[e]), e
        assert torch.equal(d1[e].float(), dh.T @ x[s]), e
        assert torch.equal(d2[e].float(), (dy[s].T @ a).bfloat16().float()), e


def test_expert_ffn_infinite_neighbours_do_not_leak():
    """An expert's rows and weights that hold inf or NaN leave the others' results alone."""
    counts = (20, 37, 5)
    x, offsets, w1, w2, dy, off = ffn_inputs(counts, 136, 72, "swiglu", 0, 77)
    clean = [t.clone() for t in (x, w1, w2, dy)]
    x[20:57], dy[20:57] = math.nan, math.inf
    w1[1], w2[1] = math.inf, math.nan
    res = []
    for t in ((x, w1, w2, dy), clean):
        leaves = [v.requires_grad_(True) for v in t[:3]]
        y = zb.expert_ffn(leaves[0], offsets, leaves[1], leaves[2])
        res.append((y, *torch.autograd.grad(y, leaves, t[3])))
    for a, b, by_rows in zip(*res, (True, True, False, False)):
        for e in (0, 2):
            s = slice(off[e], off[e + 1]) if by_rows else e
            assert torch.equal(a[s], b[s])


def test_expert_ffn_gradient_against_differences():
    """<gradient, v> against central differences of the 64-bit function along v."""
    counts = (40, 0, 23)
    for act in ("swiglu", "gelu"):
        x, offsets, w1, w2, dy, off = ffn_inputs(counts, 64, 40, act, 0, 5)
        leaves = [t.requires_grad_(True) for t in (x, w1, w2)]
        y = zb.expert_ffn(x, offsets, w1, w2, act=act)
        grads = torch.autograd.grad(y, leaves, dy)
        base = [t.detach().double() for t in leaves]
        for i in range(3):
            g = gen(60 + i)
            v = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
            eps = 1e-5

            def f(s):
                t = list(base)
                t[i] = t[i] + s * v
                return float((ffn64(t[0], off, t[1], t[2], act) * dy.double()).sum())
            diff = (f(eps) - f(-eps)) / (2 * eps)
            got = float((grads[i].double() * v).sum())
            # the gradient's elements are off by at most about 2^-7 of their norm together (near()), v has norm sqrt(numel)
            # but a random direction: 6 standard deviations of a sum of independent errors
            assert abs(got - diff) <= 6 * 2.0 ** -7 * float(grads[i].double().norm()), (act, i, got, diff)


def test_expert_ffn_survives_bad_offsets():
    """Offsets that decrease or pass the buffer end cannot reach outside of it: every kernel clamps them."""
    x, _, w1, w2, dy, _ = ffn_inputs((16, 16), 64, 64, "swiglu", 0, 1)
    leaves = [t.requires_grad_(True) for t in (x, w1, w2)]
    for off in ([5, 3, 99], [-4, 40, -1], [0, 32, 31]):
        y = zb.expert_ffn(x, torch.tensor(off, dtype=torch.int32, device="cuda"), w1, w2)
        torch.autograd.grad(y, leaves, dy)
    ops.check_waits()
    want = zb.expert_ffn(x, torch.tensor([0, 32, 32], dtype=torch.int32, device="cuda"), w1, w2)
    assert torch.equal(y, want)                # 31 after 32 counts as 32


def test_expert_ffn_partial_gradients_and_strides():
    x, offsets, w1, w2, dy, _ = ffn_inputs((30, 50), 128, 64, "swiglu", 0, 21)
    full = [t.clone().requires_grad_(True) for t in (x, w1, w2)]
    want = torch.autograd.grad(zb.expert_ffn(full[0], offsets, full[1], full[2]), full, dy)
    for i in range(3):
        t = [v.clone() for v in (x, w1, w2)]
        t[i].requires_grad_(True)
        assert torch.equal(torch.autograd.grad(zb.expert_ffn(t[0], offsets, t[1], t[2]), t[i], dy)[0], want[i])
    shifted = torch.empty(80 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(80, 128).copy_(x)
    y = zb.expert_ffn(shifted, offsets, w1.transpose(1, 2).contiguous().transpose(1, 2), w2)
    assert torch.equal(y, zb.expert_ffn(x, offsets, w1, w2))


# --------------------------------------------------------------------------------------------- norm of many, clipping
def clip64(ts, max_norm):
    total = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    return total, min(1.0, max_norm / (total + 1e-6))


@pytest.mark.parametrize("sizes", [(1,), (0, 5, 0), (3, 17, 8191, 8192, 8193, 1), (1_000_003,), tuple(range(1, 400)), (7,) * 1100])
def test_clip(sizes):
    for mixed in (False, True):
        g = gen(len(sizes))
        ts = [randn((n,), g, TYPES[i % 3] if mixed else torch.float32) for i, n in enumerate(sizes)]
        total, _ = clip64(ts, 1.0)
        # per-thread sums of at most 64 squares in fp32, then 64 bits; the root halves a relative error
        assert abs(float(zb.grad_norm(ts)) - total) <= (64 + 2) * U * total
        for limit in (0.3 * total, 3.0 * total, 0.0):
            mine = [t.clone() for t in ts]
            n = zb.clip_grad_norm_(mine, limit)
            assert abs(float(n) - total) <= 66 * U * total
            _, c = clip64(ts, limit)
            for a, b in zip(mine, ts):
                if c == 1.0:
                    assert torch.equal(a, b)
                else:
                    w = b.double() * c
                    within(a, w, (HALF[b.dtype] + 70 * U) * w.abs() + torch.finfo(b.dtype).tiny, limit)


def test_clip_range_and_special_values():
    big = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(zb.grad_norm([big])) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    small = torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(zb.grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    assert float(zb.grad_norm([torch.zeros(5, device="cuda")])) == 0.0
    t = torch.ones(100, device="cuda")
    t[7] = math.inf
    assert math.isinf(float(zb.clip_grad_norm_([t], 1.0)))
    assert bool(t[7].isnan()) and bool((t[:7] == 0).all())
    t = torch.ones(100, device="cuda", dtype=torch.bfloat16)
    t[3] = math.nan
    assert math.isnan(float(zb.clip_grad_norm_([t], 1.0))) and bool(t.isnan().all())


def test_clip_touches_nothing_else():
    """Tensors anywhere inside a buffer: what lies around them stays, byte for byte."""
    for dtype in TYPES:
        buf = randn((5000,), gen(2), dtype)
        before = buf.clone()
        parts = [buf[3:4], buf[17:1300], buf[1301:1302], buf[2001:4999]]
        zb.clip_grad_norm_(parts, 0.1)
        hit = torch.zeros(5000, dtype=torch.bool, device="cuda")
        for s in (slice(3, 4), slice(17, 1300), slice(1301, 1302), slice(2001, 4999)):
            hit[s] = True
        assert torch.equal(buf[~hit], before[~hit]) and bool((buf[hit] != before[hit]).float().mean() > 0.9)


def test_clip_orders_gaps_overlaps():
    g = gen(1)
    t = randn((30, 50), g).t()
    want = t.clone() * (1.0 / (float(t.double().norm()) + 1e-6))
    v = t._version
    zb.clip_grad_norm_([t], 1.0)
    assert torch.allclose(t, want, rtol=1e-5, atol=0) and t._version > v
    zb.clip_grad_norm_([t[:, :7]], 1.0)        # 7 columns of the transposed matrix are 7 whole rows in memory: no gaps
    for bad in ([t[:7]], [torch.ones(1, device="cuda").expand(4)], [t, t], [t, t[:, 3:]], [torch.ones(3)], [torch.ones(3, device="cuda", dtype=torch.int32)]):
        with pytest.raises(AssertionError):
            zb.clip_grad_norm_(bad, 1.0)


# ------------------------------------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("n", (2, 16, 17, 40))
def test_clip_neighbours_and_overlaps_by_count(n):
    """Short and long lists: tensors that touch are taken in any order, one shared element is refused."""
    buf = torch.ones(n * 64, device="cuda")
    parts = [buf[i * 64:(i + 1) * 64] for i in range(n)][::-1]
    parts[0] = parts[0].to(torch.bfloat16)
    parts += [buf[64:64]]                                                    # empty, inside another's span
    total = zb.clip_grad_norm_(parts, 1.0)
    # all summands are 1: sums of integers below 2^24 are exact, one rounding of the root and the type's own
    assert abs(float(total) - math.sqrt(n * 64)) <= 2 * U * math.sqrt(n * 64)
    kept = buf.clone()
    more = [torch.ones(64, device="cuda") for _ in range(n - 2)] + [buf[:64], buf[63:100]]
    with pytest.raises(AssertionError):
        zb.clip_grad_norm_(more, 1.0)
    assert torch.equal(buf, kept) and all(bool((t == 1).all()) for t in more[:-2])
    want = math.sqrt(sum(float(t.double().square().sum()) for t in more))
    # order of the kernel's sums is free: (64 n + 37) summands in fp32 at most lose one U each in the sum, half in the root
    assert abs(float(zb.grad_norm(more)) - want) <= (64 * n + 40) * U * want


def test_refusals():
    c = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i32, bf = dict(dtype=torch.int32), dict(dtype=torch.bfloat16)
    plan = ops.SortPlan(c(5, **i32), c(4, 2, **i32))
    for call in (
            lambda: zb.route_topk(c(4, 8), 9), lambda: zb.route_topk(c(4, 8), 0), lambda: zb.route_topk(c(4, 1025), 2),
            lambda: zb.route_topk(c(4, 64), 33), lambda: zb.route_topk(c(8), 2), lambda: zb.route_topk(c(4, 8, dtype=torch.float64), 2),
            lambda: zb.route_topk(c(4, 8), 2, score="relu"), lambda: zb.route_topk(c(4, 8), 2, bias=c(8)),
            lambda: zb.route_topk(c(4, 8), 2, score="sigmoid", bias=c(7)), lambda: zb.route_topk(c(4, 8), 2, score="sigmoid", bias=torch.zeros(8)),
            lambda: zb.sort_tokens(c(4, 8), c(4, 2), 4), lambda: zb.sort_tokens(c(4, 8), c(5, 2, **i32), 4),
            lambda: zb.sort_tokens(c(4, 8), c(4, 65, **i32), 4), lambda: zb.sort_tokens(c(4, 8), c(4, 2, **i32), 2049),
            lambda: zb.sort_tokens(c(4, 8), torch.zeros(4, 2, **i32), 4), lambda: zb.sort_tokens(c(4, 8), c(4, 2, **i32), 4, group_of=c(4)),
            lambda: zb.unsort_tokens(c(7, 8), plan), lambda: zb.unsort_tokens(c(8, 8), plan, c(4, 3)),
            lambda: zb.unsort_tokens(c(8, 8), plan, c(4, 2, **bf)),
            lambda: zb.expert_ffn(c(4, 16), c(3, **i32), c(2, 16, 16), c(2, 16, 8)),                         # fp32
            lambda: zb.expert_ffn(c(4, 12, **bf), c(3, **i32), c(2, 16, 12, **bf), c(2, 12, 8, **bf)),       # 12
            lambda: zb.expert_ffn(c(4, 16, **bf), c(2, **i32), c(2, 16, 16, **bf), c(2, 16, 8, **bf)),       # offsets
            lambda: zb.expert_ffn(c(4, 16, **bf), c(3, **i32), c(2, 16, 16, **bf), c(2, 16, 8, **bf), act="gelu"),
            lambda: zb.expert_ffn(c(4, 16, **bf), c(3, dtype=torch.int64), c(2, 16, 16, **bf), c(2, 16, 8, **bf))):
        with pytest.raises(AssertionError):
            call()


# -------------------------------------------------------------------------------- together, streams, captured graphs
def small_layer(act="swiglu", redundant=2):
    from zepp_b200 import workloads as wl
    from zepp_b200.layer import LocalGroup
    shape = zb.ModelShape(16, 4, 256, 128, act=act)
    cfg = zb.EPMoEConfig(shape=shape, ranks=1, ranks_per_node=1, max_tokens_per_rank=64, redundant_slots_per_rank=redundant)
    g = torch.Generator().manual_seed(0)
    ids, _ = wl.routing(1, 64, 4, wl.popularity(16, 1.0, g), g)
    layer = zb.EPMoE(cfg, LocalGroup(0, 1), ids, ids)
    W1 = torch.stack([wl.expert_w1(e, shape) for e in range(16)]).cuda()
    W2 = torch.stack([wl.expert_w2(e, shape) for e in range(16)]).cuda()
    layer.load_weights(lambda e: W1[e], lambda e: W2[e])
    return layer, shape, W1, W2


def test_layer_gate_feeds_the_step_and_pads_stay_pads():
    layer, shape, W1, W2 = small_layer()
    g = gen(3)
    logits, x = randn((64, 16), g), randn((64, 256), g, torch.bfloat16)
    logits[60:] = -math.inf                                     # a padded batch
    ids, w = layer.gate(logits)
    assert bool((ids[60:] == -1).all())
    y = layer.step(ids, w, x).clone()
    layer.check()
    y2 = layer.forward_train(x, ids, w)
    assert bool((y[60:] == 0).all()) and bool((y2[60:] == 0).all())
    near(y2[:60], y[:60], "step and forward_train")
    layer.close()


@pytest.mark.parametrize("act", ["swiglu", "gelu"])
def test_training_step_of_a_layer(act):
    """gate -> sort -> products -> back, all gradients, clipping, an update in place that the next step() sees."""
    layer, shape, W1, W2 = small_layer(act)
    g = gen(8)
    n, E = 90, shape.num_experts
    x = randn((n, 256), g, torch.bfloat16).requires_grad_(True)
    router = randn((E, 256), g, std=256 ** -0.5).requires_grad_(True)
    dy = randn((n, 256), g, torch.bfloat16)
    w1, w2 = layer.train_weights()
    ids, w = layer.gate(x.float() @ router.T)
    y = layer.forward_train(x, ids, w)
    y.backward(dy)
    m = [t.detach().double().requires_grad_(True) for t in (x, router, W1, W2)]
    ids64, w64 = gate64(m[0] @ m[1].T, 4, "softmax", True, None, 1.0)
    same = (ids64 == ids).all(1)                               # a product in fp32 may order two near-equal logits otherwise
    assert int((~same).sum()) == 0
    y64 = torch.zeros((n, 256), dtype=torch.float64, device="cuda")
    for e in range(E):
        t, k = (ids64 == e).nonzero(as_tuple=True)
        out = act64(m[0][t] @ m[2][e].T, act, shape.ffn_hidden) @ m[3][e].T
        y64 = y64.index_add(0, t, out * w64[t, k, None])
    near(y.detach(), y64.detach(), "y")
    g64 = torch.autograd.grad(y64, m, dy.double())
    near(x.grad, g64[0], "dx")
    near(router.grad, g64[1], "drouter")
    slot = (1 + layer.placement.l2p[:, 0]).long().cuda()
    near(w1.grad[slot], g64[2], "dw1")
    near(w2.grad[slot], g64[3], "dw2")
    rest = torch.ones(w1.shape[0], dtype=torch.bool, device="cuda")
    rest[slot] = False
    assert bool((w1.grad[rest] == 0).all()) and bool((w2.grad[rest] == 0).all())
    total = math.sqrt(sum(float(t.grad.double().square().sum()) for t in (w1, w2, router)))
    norm = layer.clip_grad_norm_(total / 2, others=[router])
    assert abs(float(norm) - total) <= 1e-5 * total
    left = math.sqrt(sum(float(t.grad.double().square().sum()) for t in (w1, w2, router)))
    assert abs(left - total / 2) <= 2.0 ** -8 * total / 2
    with torch.no_grad():
        for p in (w1, w2):
            p.add_(p.grad, alpha=-0.5)
    layer.set_tokens(64)
    ids64t, wt = ids[:64].contiguous(), w.detach()[:64].contiguous()
    with torch.no_grad():
        y_train = layer.forward_train(x[:64], ids64t, wt)
        y_step = layer.step(ids64t, wt, x.detach()[:64].contiguous())
    layer.check()
    near(y_train, y_step, "after the update")
    layer.close()


def test_forward_train_refuses_what_it_cannot_do():
    layer, shape, _, _ = small_layer()
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    ids, w = torch.zeros(4, 4, dtype=torch.int32, device="cuda"), torch.zeros(4, 4, device="cuda")
    with pytest.raises(AssertionError):
        layer.forward_train(x[:3], ids, w)
    with pytest.raises(AssertionError):
        layer.gate(torch.zeros(4, 15, device="cuda"))
    for changed in (dict(ranks=2, ranks_per_node=2), dict(swap=True)):
        keep, layer.cfg = layer.cfg, dataclasses.replace(layer.cfg, **changed)
        with pytest.raises(AssertionError):
            layer.forward_train(x, ids, w)
        layer.cfg = keep
    layer.close()


def whole(s):
    ids, w = zb.route_topk(s["logits"], 4)
    rows, plan = zb.sort_tokens(s["x"], ids, 8)
    rows = zb.expert_ffn(rows, plan.offsets, s["w1"], s["w2"])
    y = zb.unsort_tokens(rows, plan, w)
    grads = torch.autograd.grad(y, (s["logits"], s["x"], s["w1"], s["w2"]), s["dy"])
    norm = zb.clip_grad_norm_(grads, 0.5)
    return [ids, w, plan.offsets, plan.position, y, *grads, norm]


def whole_state(seed, T=40):
    g = gen(seed)
    s = dict(logits=randn((T, 8), g), x=randn((T, 128), g, torch.bfloat16), w1=randn((8, 128, 128), g, torch.bfloat16, 0.1),
             w2=randn((8, 128, 64), g, torch.bfloat16, 0.1))
    for t in s.values():
        t.requires_grad_(True)
    return dict(s, dy=randn((T, 128), g, torch.bfloat16))


def test_same_bits_twice_on_another_stream_and_in_two_graphs():
    states = [whole_state(1), whole_state(2, T=3000)]
    want = [[t.detach().clone() for t in whole(s)] for s in states]
    for s, w in zip(states, want):
        assert all(torch.equal(a, b) for a, b in zip(whole(s), w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = whole(states[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    # two graphs out of one memory pool, replayed in turn with new inputs
    del got
    statics = [{k: v.detach().clone().requires_grad_(v.requires_grad) for k, v in s.items()} for s in states]
    graphs, outs = [], []
    for s in statics:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(whole(s))
        graphs.append(graph)
    fresh = [whole_state(11), whole_state(12, T=3000)]
    wants = [[t.detach().clone() for t in whole(s)] for s in fresh]
    for order in ((0, 1), (1, 0)):
        for i in order:
            with torch.no_grad():
                for k in statics[i]:
                    statics[i][k].copy_(fresh[i][k])
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], wants[i])), (order, i)
    ops.check_waits()


def test_calls_on_two_streams_at_once():
    states = [whole_state(21, T=700), whole_state(22, T=900)]
    want = [[t.detach().clone() for t in whole(s)] for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = whole(states[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_sort_of_many_copies_passes_32_bit_offsets():
    """Rows beyond 2^31 bytes and elements: 70,000 tokens x 8 copies x 4096 elements are 2.29e9 elements."""
    T, K, H = 70_000, 8, 4096
    g = gen(1)
    ids = torch.randint(0, 64, (T, K), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randint(-100, 100, (T, H), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    rows, plan = zb.sort_tokens(x, ids, 64)
    assert int(plan.offsets[-1]) == T * K
    last = (plan.position == T * K - 1).nonzero()[0]
    assert torch.equal(rows[T * K - 1], x[last[0]])
    some = torch.randint(0, T, (500,), generator=g, device="cuda")
    assert torch.equal(rows[plan.position[some].long()], x[some][:, None, :].expand(-1, K, -1))
    y = zb.unsort_tokens(rows, plan, torch.full((T, K), 0.125, device="cuda"))
    assert torch.equal(y, x)


@pytest.mark.parametrize("T, K, H, dtype", [(700, 8, 2048, torch.bfloat16), (613, 3, 1032, torch.float32), (2500, 11, 1160, torch.float16), (601, 20, 7168, torch.bfloat16)])
def test_unsort_of_many_long_rows(T, K, H, dtype):
    """Long rows in large numbers go through shared memory in pieces: whole and ragged last pieces, more copies than eight."""
    g = gen(T)
    ids = torch.randint(-2, 50, (T, K), generator=g, device="cuda", dtype=torch.int32)
    ids[5] = -1
    _, plan = zb.sort_tokens(randn((T, 8), g), ids, 50)
    r, w = randn((T * K, H), g, dtype).requires_grad_(True), randn((T, K), g).requires_grad_(True)
    dy = randn((T, H), g, dtype)
    y = zb.unsort_tokens(r, plan, w)
    dr, dw = torch.autograd.grad(y, (r, w), dy)
    took = (plan.position >= 0)
    pos = plan.position.clamp_min(0).long()
    y64, size, dw64, dsize = (torch.zeros((T, n), dtype=torch.float64, device="cuda") for n in (H, H, K, K))
    dr64 = torch.zeros((T * K, H), dtype=torch.float64, device="cuda")
    for k in range(K):
        row = r.detach()[pos[:, k]].double() * took[:, k, None]
        y64 += row * w.detach()[:, k, None].double()
        size += (row * w.detach()[:, k, None].double()).abs()
        dw64[:, k], dsize[:, k] = (row * dy.double()).sum(1), (row * dy.double()).abs().sum(1)
        t = took[:, k].nonzero()[:, 0]
        dr64[pos[t, k]] = w.detach()[t, k, None].double() * dy[t].double()
    within(y, y64, HALF[dtype] * y64.abs() + 2 * K * U * size + torch.finfo(dtype).tiny, "y")
    within(dr, dr64, (HALF[dtype] + 2 * U) * dr64.abs() + torch.finfo(dtype).tiny, "drows")
    within(dw, dw64, (H / 32 + 8 + 13) * U * dsize + 1e-30, "dweights")
    assert torch.equal(torch.autograd.grad(zb.unsort_tokens(r, plan, w.detach()), r, dy)[0], dr)       # without dweights
    assert torch.equal(torch.autograd.grad(zb.unsort_tokens(r.detach(), plan, w), w, dy)[0], dw)       # without drows
    ops.check_waits()


def test_expert_ffn_without_rows():
    w1, w2 = randn((3, 32, 24), gen(1), torch.bfloat16), randn((3, 24, 16), gen(1), torch.bfloat16)
    leaves = [torch.zeros((0, 24), dtype=torch.bfloat16, device="cuda"), w1, w2]
    for t in leaves:
        t.requires_grad_(True)
    y = zb.expert_ffn(leaves[0], torch.zeros(4, dtype=torch.int32, device="cuda"), w1, w2)
    assert y.shape == (0, 24)
    dx, d1, d2 = torch.autograd.grad(y, leaves, torch.zeros_like(y))
    assert dx.shape == (0, 24) and d1.shape == w1.shape and not d1.any() and not d2.any()


def test_gradients_are_first_derivatives_only():
    """With create_graph the gradients come out the same; a second derivative is an error, not a wrong number."""
    l = randn((5, 16), gen(2)).requires_grad_(True)
    w = zb.route_topk(l, 3)[1]
    once = torch.autograd.grad(w.square().sum(), l, retain_graph=True)[0]
    twice = torch.autograd.grad(w.square().sum(), l, create_graph=True)[0]
    assert torch.equal(once, twice)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(twice.sum(), l)


def test_padded_batch_through_the_whole_chain():
    """Pad rows (logits masked out) cost nothing and change nothing: the real tokens' results are those of the batch without
    them, and pad tokens get zeros, in both directions."""
    T, pads, G, H, I, K = 70, 26, 12, 128, 72, 3
    g = gen(31)
    logits, x = randn((T, G), g), randn((T, H), g, torch.bfloat16)
    w1, w2 = randn((G, 2 * I, H), g, torch.bfloat16, 0.1), randn((G, H, I), g, torch.bfloat16, 0.1)
    dy = randn((T, H), g, torch.bfloat16)
    res = []
    for n in (0, pads):
        l = torch.cat([logits, torch.full((n, G), -math.inf, device="cuda")]).requires_grad_(True)
        xs = torch.cat([x, torch.full((n, H), math.nan, dtype=torch.bfloat16, device="cuda")]).requires_grad_(True)
        a, b = w1.clone().requires_grad_(True), w2.clone().requires_grad_(True)
        ids, w = zb.route_topk(l, K, renormalize=False)
        rows, plan = zb.sort_tokens(xs, ids, G)
        y = zb.unsort_tokens(zb.expert_ffn(rows, plan.offsets, a, b), plan, w)
        d = torch.cat([dy, torch.full((n, H), math.nan, dtype=torch.bfloat16, device="cuda")])
        gl, gx, ga, gb = torch.autograd.grad(y, (l, xs, a, b), d)
        assert not y[T:].any() and not gl[T:].any() and not gx[T:].any()
        res.append((y[:T], gl[:T], gx[:T], ga, gb))
    for u, v in zip(*res):
        assert torch.equal(u, v)


def test_calls_of_every_kind_of_argument():
    """Gradients through what is optional or copied on the way: no weights, transposed weights, generators, views."""
    g = gen(41)
    ids = torch.randint(-1, 5, (30, 3), generator=g, device="cuda", dtype=torch.int32)
    _, plan = zb.sort_tokens(randn((30, 16), g), ids, 5)
    r = randn((90, 16), g).requires_grad_(True)
    dy = randn((30, 16), g)
    dr = torch.autograd.grad(zb.unsort_tokens(r, plan), r, dy)[0]
    want = torch.zeros(90, 16, device="cuda")
    t, k = (plan.position >= 0).nonzero(as_tuple=True)
    want[plan.position[t, k].long()] = dy[t]
    assert torch.equal(dr, want)
    # weights held the other way round: the gradient comes back in their layout
    x, offsets, w1, w2, d, _ = ffn_inputs((20, 30), 64, 40, "swiglu", 0, 42)
    flip = w1.transpose(1, 2).contiguous().requires_grad_(True)
    plain = w1.clone().requires_grad_(True)
    a = torch.autograd.grad(zb.expert_ffn(x, offsets, flip.transpose(1, 2), w2), flip, d)[0]
    b = torch.autograd.grad(zb.expert_ffn(x, offsets, plain, w2), plain, d)[0]
    assert torch.equal(a, b.transpose(1, 2))
    # a part of a longer buffer, and every other offset of a table
    wide = torch.stack([offsets, offsets], 1)
    assert torch.equal(zb.expert_ffn(torch.cat([x, x])[:50], wide[:, 0], w1, w2), zb.expert_ffn(x, offsets, w1, w2))
    ts = [randn((7,), g), randn((), g)]
    before = [t.clone() for t in ts]
    n = zb.clip_grad_norm_((t for t in ts), math.inf)
    assert all(torch.equal(u, v) for u, v in zip(ts, before)) and float(n) > 0
    with torch.inference_mode():
        w = zb.route_topk(randn((4, 8), g), 2)[1]
        assert torch.allclose(w.sum(1), torch.ones(4, device="cuda"), atol=1e-6)
        zb.clip_grad_norm_([torch.ones(4, device="cuda")], 1.0)
