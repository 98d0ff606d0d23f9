"""The operators around the expert-parallel layer as measured calls: the gate, tokens sorted by expert and back, the experts' products,
and the norm of all gradients with clipping, each with its gradient where it has one.

`own` chooses between the plain forms (elementary torch operations in 32 bits) and this package's kernels.
"""
import math

import torch

own = False


# ---------------------------------------------------------------------------------------------------------------------------- cases
def _gate(name, tokens, experts, k, score, renormalize, bias, dtype, train, masked=0.0):
    c = dict(op="gate", tokens=tokens, experts=experts, k=k, score=score, renormalize=renormalize, bias=bias, dtype=dtype,
             train=train, masked=masked)
    return dict(c, name=name) if name else c


def _sort(name, tokens, k, experts, hidden, dtype, train, pads=0.0):
    c = dict(op="sort", tokens=tokens, k=k, experts=experts, hidden=hidden, dtype=dtype, train=train, pads=pads)
    return dict(c, name=name) if name else c


def _ffn(name, rows, experts, hidden, ffn, act, train, skew=0.0, spare=0):
    c = dict(op="ffn", rows=rows, experts=experts, hidden=hidden, ffn=ffn, act=act, train=train, skew=skew, spare=spare)
    return dict(c, name=name) if name else c


def _clip(name, tensors, elements, dtype, clips):
    c = dict(op="clip", tensors=tensors, elements=elements, dtype=dtype, clips=clips)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the gate of one decode step of a serving batch (128 experts, top-8 renormalised softmax, fp32 logits)
        _gate("gate decode", 16, 128, 8, "softmax", True, False, "float32", False),
        # a training batch of a 384-expert layer: sigmoid scores, a balancing bias that takes part in the choice only, bf16 logits
        _gate("gate train sigmoid bias", 16381, 384, 8, "sigmoid", True, True, "bfloat16", True),
        # softmax over all experts without renormalising; some experts masked out, some rows masked out altogether (padded batch)
        _gate("gate train softmax masked", 8192, 128, 8, "softmax", False, False, "float32", True, masked=0.05),
        # one decode step: 32 tokens to 8 of 128 experts and back
        _sort("sort decode", 32, 8, 128, 2048, "bfloat16", False),
        # a training micro-batch with gradients, 4096 wide rows
        _sort("sort train", 8192, 8, 128, 4096, "bfloat16", True),
        # fp32 rows of an odd width, top-6, a tenth of the copies pads
        _sort("sort train odd fp32", 1531, 6, 160, 1003, "float32", True, pads=0.1),
        # decode: 8 tokens x top-8, most experts idle; bound by the weights of those that have a row
        _ffn("ffn decode", 64, 128, 2048, 768, "swiglu", False),
        # a training micro-batch of 4096 tokens x top-8 on the 128-expert layer of 2048 / 768
        _ffn("ffn train 128 experts", 32768, 128, 2048, 768, "swiglu", True, skew=0.5),
        # one rank's share of a wide layer (7168 / 2048), uneven experts, some without rows, a buffer longer than its rows
        _ffn("ffn train wide", 3001, 12, 7168, 2048, "swiglu", True, skew=1.5, spare=77),
        # GELU experts of sizes off every tile
        _ffn("ffn train odd gelu", 333, 7, 392, 136, "gelu", True, skew=1.0, spare=5),
        # the gradients of a model's small parameters: many tensors, odd lengths, fp32, this step is not clipped
        _clip("clip many small", 240, 2_000_003, "float32", False),
        # the bf16 gradients of a 128-expert layer's weights, clipped
        _clip("clip experts", 3, 604_241_920, "bfloat16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gate", "sort", "ffn", "clip"))
    if op == "gate":
        experts = rng.choice((rng.randint(9, 64), 64, 128, 160, 256, 384, rng.randint(65, 512)))
        score = rng.choice(("softmax", "sigmoid"))
        return _gate(None, _log(rng, 1, 16000), experts, rng.randint(1, min(10, experts)), score, rng.random() < 0.6,
                     score == "sigmoid" and rng.random() < 0.6, rng.choice(("float32", "bfloat16", "float16")),
                     rng.random() < 0.6, masked=rng.choice((0.0, 0.0, 0.1)))
    if op == "sort":
        hidden = rng.choice((2048, 4096, 7168, 8 * rng.randint(8, 512), rng.randint(65, 4000)))
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        k = rng.randint(1, 10)
        most = 8192 * 8 * 4096 * 2 // (hidden * k * (4 if dtype == "float32" else 2))
        return _sort(None, _log(rng, 1, min(8192, most)), k, rng.choice((8, 60, 128, 256, 384, rng.randint(2, 512))), hidden,
                     dtype, rng.random() < 0.6, pads=rng.choice((0.0, 0.0, 0.2)))
    if op == "ffn":
        hidden, ffn = rng.choice(((2048, 768), (2048, 768), (4096, 1024), (1024, 512), (8 * rng.randint(20, 320), 8 * rng.randint(8, 160))))
        experts = rng.choice((8, 16, 60, rng.randint(1, 128)))
        if experts * hidden * ffn > 128 * 2048 * 768:
            experts = 128 * 2048 * 768 // (hidden * ffn)
        return _ffn(None, _log(rng, 1, min(32768, 32768 * 2048 * 768 // (hidden * ffn))), experts, hidden, ffn,
                    rng.choice(("swiglu", "swiglu", "gelu")), rng.random() < 0.6, skew=rng.choice((0.0, 0.5, 1.0)),
                    spare=rng.choice((0, rng.randint(1, 200))))
    tensors = _log(rng, 1, 400)
    return _clip(None, tensors, _log(rng, 1000 + tensors, 300_000_000), rng.choice(("bfloat16", "float32", "float16", "mixed")),
                 rng.random() < 0.7)


# --------------------------------------------------------------------------------------------------------------------------- inputs
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SCALE = 2.5        # the factor that sigmoid gates commonly put on their weights


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _sizes(case):
    """Lengths of the clip case's tensors: uneven, odd ones among them, `elements` in all (or as near as the spread allows)."""
    n, total = case["tensors"], case["elements"]
    if n == 1:
        return [total]
    share = [1.0 + (7 * i % 11) for i in range(n)]
    cut = [max(1, int(total * s / sum(share))) for s in share]
    cut[-1] = max(1, cut[-1] + total - sum(cut))
    return cut


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "gate":
        T, G, k = case["tokens"], case["experts"], case["k"]
        logits = _randn((T, G), g, std=1.5)
        if case["masked"]:
            logits.masked_fill_(torch.rand((T, G), generator=g, device="cuda") < case["masked"], -math.inf)
            logits.masked_fill_(torch.rand((T, 1), generator=g, device="cuda") < case["masked"], -math.inf)
        logits = logits.to(_TYPES[case["dtype"]]).requires_grad_(case["train"])
        return dict(case=case, logits=logits, bias=_randn((G,), g, std=0.05) if case["bias"] else None, dw=_randn((T, k), g),
                    scale=_SCALE if case["score"] == "sigmoid" else 1.0)
    if op == "sort":
        T, K, G, H, t = case["tokens"], case["k"], case["experts"], case["hidden"], _TYPES[case["dtype"]]
        # K distinct experts for each token where there are that many, some experts more popular than others
        liking = _randn((G,), g, std=0.7) + _randn((T, G), g)
        ids = liking.topk(min(K, G), dim=1).indices
        ids = torch.cat([ids] * -(-K // ids.shape[1]), 1)[:, :K].int()
        if case["pads"]:
            ids = torch.where(torch.rand((T, K), generator=g, device="cuda") < case["pads"], torch.full_like(ids, -1), ids)
        s = dict(case=case, ids=ids.contiguous(), x=_randn((T, H), g, t).requires_grad_(case["train"]),
                 rows=_randn((T * K, H), g, t).requires_grad_(case["train"]),
                 w=torch.softmax(_randn((T, K), g), 1).requires_grad_(case["train"]))
        if case["train"]:
            s.update(dy=_randn((T, H), g, t), dsorted=_randn((T * K, H), g, t))
        return s
    if op == "ffn":
        M, G, H, I = case["rows"], case["experts"], case["hidden"], case["ffn"]
        f1 = (2 if case["act"] == "swiglu" else 1) * I
        host = torch.Generator().manual_seed(int(seed))
        p = (torch.arange(G, dtype=torch.float64) + 1.0).pow(-case["skew"])[torch.randperm(G, generator=host)]
        counts = torch.bincount(torch.multinomial(p, M, replacement=True, generator=host), minlength=G)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
        n = M + case["spare"]
        s = dict(case=case, offsets=offsets.int().cuda(), most=int(counts.max()), rows=_randn((n, H), g, torch.bfloat16),
                 w1=_randn((G, f1, H), g, torch.bfloat16, H ** -0.5), w2=_randn((G, H, I), g, torch.bfloat16, I ** -0.5))
        if case["train"]:
            s["dy"] = _randn((n, H), g, torch.bfloat16)
            for name in ("rows", "w1", "w2"):
                s[name].requires_grad_(True)
        return s
    order = ("bfloat16", "float32", "float16")
    sizes = _sizes(case)
    names = [order[i % 3] if case["dtype"] == "mixed" else case["dtype"] for i in range(len(sizes))]
    # the gradients lie one behind the other in a buffer for each type, as a training program's buckets hold them
    flat = {t: _randn((sum(n for n, m in zip(sizes, names) if m == t),), g, _TYPES[t], 0.01) for t in dict.fromkeys(names)}
    parts = {t: iter(flat[t].split([n for n, m in zip(sizes, names) if m == t])) for t in flat}
    total = math.sqrt(sum(sizes)) * 0.01
    return dict(case=case, grads=[next(parts[t]) for t in names], flat=list(flat.values()),
                max_norm=total * (0.25 if case["clips"] else 4.0))


# ---------------------------------------------------------------------------------------------------------------------- plain forms
def _plain_gate(s):
    case = s["case"]
    G, k, scale = case["experts"], case["k"], s["scale"]
    l = s["logits"].float()
    softmax = case["score"] == "softmax"
    # the choice is by values next to a border: in 64 bits
    key = l.double()
    if s["bias"] is not None:
        key = torch.where(key == -math.inf, key, 1.0 / (1.0 + torch.exp(-key)) + s["bias"].double())
    best, ids = torch.sort(key, dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    found = best > -math.inf
    if softmax:
        top = l.amax(1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
        p = torch.exp(l - top)
        if not case["renormalize"]:
            p = p / p.sum(1, keepdim=True).clamp_min(1e-30)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    chosen = torch.where(found, p.gather(1, ids), torch.zeros((), device=l.device))
    if case["renormalize"]:
        total = chosen.sum(1, keepdim=True) + 1e-20
        w = scale * chosen / total
    else:
        w = scale * chosen
    out = [torch.where(found, ids, torch.full_like(ids, -1)).int(), w]
    if case["train"]:
        dw = torch.where(found, s["dw"], torch.zeros((), device=l.device)) * scale
        if case["renormalize"]:
            dp = (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
        else:
            dp = dw
        if softmax and not case["renormalize"]:
            dl = -p * (dp * chosen).sum(1, keepdim=True)
            dl = dl.scatter_add(1, ids, dp * chosen)
        else:
            slope = chosen if softmax else chosen * (1.0 / (1.0 + torch.exp(l.gather(1, ids))))
            dl = torch.zeros_like(l).scatter_add(1, ids, torch.where(found, dp * slope, torch.zeros((), device=l.device)))
        out.append(dl.to(s["logits"].dtype))
    return out


def _plain_sort(s):
    case = s["case"]
    T, K, G, H = case["tokens"], case["k"], case["experts"], case["hidden"]
    n = T * K
    ids = s["ids"].reshape(-1).long()
    key = torch.where(ids < 0, torch.full_like(ids, G), ids)
    key, order = torch.sort(key, stable=True)
    at = torch.empty_like(order)
    at[order] = torch.arange(n, device=order.device)
    position = torch.where(ids < 0, torch.full_like(at, -1), at)
    offsets = (key[None, :] < torch.arange(G + 1, device=key.device)[:, None]).sum(1).int()
    alive = (key < G)[:, None]
    rows = torch.where(alive, s["x"][order // K], torch.zeros((), dtype=s["x"].dtype, device=key.device))
    took = (position >= 0).view(T, K)
    pick = position.clamp_min(0)
    w = torch.where(took, s["w"], torch.zeros((), device=key.device))
    y = (s["rows"][pick].float().view(T, K, H) * w[..., None]).sum(1).to(s["x"].dtype)
    out = [rows, offsets, position.view(T, K).int(), y]
    if case["train"]:
        dx = (s["dsorted"][pick].float().view(T, K, H) * took[..., None]).sum(1).to(s["x"].dtype)
        dy = s["dy"].float()
        drows = torch.where(alive, dy[order // K] * s["w"].reshape(-1)[order][:, None], torch.zeros((), device=key.device))
        dw = (s["rows"][pick].float().view(T, K, H) * dy[:, None, :]).sum(2) * took
        out += [dx, drows.to(s["x"].dtype), dw]
    return out


def _plain_ffn(s):
    case = s["case"]
    G, I, R = case["experts"], case["ffn"], s["most"]
    off = s["offsets"].long()
    n = s["rows"].shape[0]
    # every expert's rows in a block of its own, zero behind its last row
    place = off[:-1, None] + torch.arange(R, device=off.device)[None, :]
    real = place < off[1:, None]
    place = place.clamp_max(n - 1)
    x = s["rows"].float()[place] * real[..., None]
    w1, w2 = s["w1"].float(), s["w2"].float()

    r = torch.arange(n, device=off.device)
    expert = (r[:, None] >= off[None, 1:]).sum(1)
    block_row = (expert * R + r - off[expert.clamp_max(G)]).clamp_max(G * R - 1)

    def back(blocks):
        out = blocks.view(G * R, -1)[block_row] * (expert < G)[:, None]
        return out.bfloat16()

    h = torch.bmm(x, w1.transpose(1, 2))
    if case["act"] == "swiglu":
        gate, up = h[..., :I], h[..., I:]
        sig = 1.0 / (1.0 + torch.exp(-gate))
        a = gate * sig * up
    else:
        cdf = 0.5 * (1.0 + torch.erf(h * 0.5 ** 0.5))
        a = h * cdf
    out = [back(torch.bmm(a, w2.transpose(1, 2)))]
    if case["train"]:
        dy = s["dy"].float()[place] * real[..., None]
        da = torch.bmm(dy, w2)
        if case["act"] == "swiglu":
            dh = torch.cat([da * up * sig * (1.0 + gate * (1.0 - sig)), da * gate * sig], 2)
        else:
            dh = da * (cdf + h * torch.exp(-0.5 * h * h) * (2.0 * math.pi) ** -0.5)
        out += [back(torch.bmm(dh, w1)), torch.bmm(dh.transpose(1, 2), x).bfloat16(), torch.bmm(dy.transpose(1, 2), a).bfloat16()]
    return out


def _plain_clip(s):
    grads = s["grads"]
    total = torch.stack([t.float().square().sum() for t in grads]).sum().sqrt()
    c = (s["max_norm"] / (total + 1e-6)).clamp_max(1.0)
    [t.copy_(t.float() * c) for t in grads]
    return [total] + s["flat"]


# ------------------------------------------------------------------------------------------------------------ this package's kernels
def _own_run(s):
    import zepp_b200 as zb
    case, op = s["case"], s["case"]["op"]
    if op == "gate":
        ids, w = zb.route_topk(s["logits"], case["k"], score=case["score"], renormalize=case["renormalize"], bias=s["bias"],
                               scale=s["scale"])
        if not case["train"]:
            return [ids, w]
        return [ids, w, torch.autograd.grad(w, s["logits"], s["dw"])[0]]
    if op == "sort":
        rows, plan = zb.sort_tokens(s["x"], s["ids"], case["experts"])
        y = zb.unsort_tokens(s["rows"], plan, s["w"])
        out = [rows, plan.offsets, plan.position, y]
        if case["train"]:
            out.append(torch.autograd.grad(rows, s["x"], s["dsorted"])[0])
            out.extend(torch.autograd.grad(y, (s["rows"], s["w"]), s["dy"]))
        return out
    if op == "ffn":
        y = zb.expert_ffn(s["rows"], s["offsets"], s["w1"], s["w2"], act=case["act"])
        if not case["train"]:
            return [y]
        return [y, *torch.autograd.grad(y, (s["rows"], s["w1"], s["w2"]), s["dy"])]
    return [zb.clip_grad_norm_(s["grads"], s["max_norm"]), *s["flat"]]


_PLAIN = {"gate": _plain_gate, "sort": _plain_sort, "ffn": _plain_ffn, "clip": _plain_clip}


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "gate":
        e = 4 if case["dtype"] == "float32" else 2
        n = case["tokens"] * case["experts"]
        chosen = case["tokens"] * case["k"]
        b = n * e + 8 * chosen
        if case["train"]:
            b += n * e + 4 * chosen         # the gradient is as large as the logits; the given gradient of the weights
        return {"bytes": b, "flops": 8 * n * (2 if case["train"] else 1)}
    if op == "sort":
        e = 4 if case["dtype"] == "float32" else 2
        T, K, H = case["tokens"], case["k"], case["hidden"]
        there = T * H * e * (1 + K)
        b = 2 * there + T * K * 12 + 4 * (case["experts"] + 1)
        f = 2 * T * K * H
        if case["train"]:
            b += there + T * H * e * (1 + K) + T * K * 4      # dx from its rows; dy read and drows written (the rows are read above)
            f += 4 * T * K * H
        return {"bytes": b, "flops": f}
    if op == "ffn":
        M, G, H, I = case["rows"], case["experts"], case["hidden"], case["ffn"]
        f1 = (2 if case["act"] == "swiglu" else 1) * I
        active = G * (1.0 - (1.0 - 1.0 / G) ** M)             # experts that have a row, for evenly spread rows
        weights = 2 * (f1 * H + H * I)
        b = int(active * weights) + 2 * (2 * M * H)
        f = 2 * M * (f1 * H + H * I)
        if case["train"]:
            b += G * weights + 2 * (2 * M * H)                # gradients of all weights; dy read, the rows' gradient written
            f *= 3
        return {"bytes": b, "flops": f}
    sizes, e = _sizes(case), {"float32": 4, "bfloat16": 2, "float16": 2}
    order = ("bfloat16", "float32", "float16")
    b = sum(n * e[order[i % 3] if case["dtype"] == "mixed" else case["dtype"]] for i, n in enumerate(sizes))
    return {"bytes": b * (2 if case["clips"] else 1), "flops": 3 * sum(sizes)}


# ---------------------------------------------------------------------------------------------------------------------------- exact
def _exact_gate(s):
    case = s["case"]
    T, G, k = case["tokens"], case["experts"], case["k"]
    l = s["logits"].detach().double()
    score = l.clone()
    if s["bias"] is not None:
        score = torch.sigmoid(l) + s["bias"].double()
        score[l == -math.inf] = -math.inf
    ids = torch.full((T, k), -1, dtype=torch.int64, device=l.device)
    left = score.clone()
    index = torch.arange(G, device=l.device).expand(T, G)
    for j in range(k):                                        # one after the other: the largest left, the lowest index among equals
        top = left.max(1, keepdim=True).values
        first = torch.where(left == top, index, G).min(1).values
        some = top[:, 0] > -math.inf
        ids[some, j] = first[some]
        left[torch.arange(T, device=l.device), first] = -math.inf
    mask = torch.zeros((T, G), dtype=torch.float64, device=l.device)
    mask.scatter_add_(1, ids.clamp_min(0), (ids >= 0).double())
    with torch.enable_grad():
        z = l.clone().requires_grad_(True)
        if case["score"] == "softmax":
            alive = torch.where((l > -math.inf).any(1, keepdim=True), z, torch.zeros_like(z))
            p = torch.softmax(alive, 1)
        else:
            p = torch.sigmoid(z)
        if case["renormalize"]:
            total = (p * mask).sum(1, keepdim=True)
            p = p / torch.where(total > 0, total, torch.ones_like(total))
        w = s["scale"] * p.gather(1, ids.clamp_min(0)) * (ids >= 0)
        out = [ids.int(), w.detach()]
        if case["train"]:
            dl = torch.autograd.grad(w, z, s["dw"].double())[0]
            out.append(torch.where(l > -math.inf, dl, torch.zeros_like(dl)))
    return out


def _exact_sort(s):
    case = s["case"]
    T, K, G, H = case["tokens"], case["k"], case["experts"], case["hidden"]
    ids = s["ids"].reshape(-1).long()
    counts = torch.bincount(ids[ids >= 0], minlength=G)
    offsets = torch.zeros(G + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = counts.cumsum(0)
    position = torch.full((T * K,), -1, dtype=torch.int64, device=ids.device)
    for e in range(G):
        mine = (ids == e).nonzero()[:, 0]
        position[mine] = offsets[e] + torch.arange(mine.numel(), device=ids.device)
    rows = torch.zeros((T * K, H), dtype=torch.float64, device=ids.device)
    pos2 = position.view(T, K)
    y = torch.zeros((T, H), dtype=torch.float64, device=ids.device)
    w = s["w"].detach().double()
    x, r = s["x"].detach(), s["rows"].detach()
    extra = [torch.zeros_like(y), torch.zeros_like(rows), torch.zeros((T, K), dtype=torch.float64, device=ids.device)] if case["train"] else []
    for k in range(K):
        t = (pos2[:, k] >= 0).nonzero()[:, 0]
        p = pos2[t, k]
        rows[p] = x[t].double()
        y[t] += w[t, k, None] * r[p].double()
        if extra:
            dy = s["dy"][t].double()
            extra[0][t] += s["dsorted"][p].double()
            extra[1][p] = w[t, k, None] * dy
            extra[2][t, k] = (dy * r[p].double()).sum(1)
    return [rows, offsets.int(), pos2.int(), y] + extra


def _exact_ffn(s):
    case = s["case"]
    I, train = case["ffn"], case["train"]
    off = s["offsets"].tolist()
    rows, w1, w2 = s["rows"].detach(), s["w1"].detach(), s["w2"].detach()
    wide = dict(dtype=torch.float64, device=rows.device)
    y = torch.zeros(rows.shape, **wide)
    if train:
        dx, d1, d2 = torch.zeros(rows.shape, **wide), torch.zeros(w1.shape, **wide), torch.zeros(w2.shape, **wide)
    for e in range(case["experts"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        x, a1, a2 = rows[lo:hi].double(), w1[e].double(), w2[e].double()
        h = x @ a1.T
        if case["act"] == "swiglu":
            sig = torch.sigmoid(h[:, :I])
            a = h[:, :I] * sig * h[:, I:]
        else:
            a = h * torch.special.ndtr(h)
        y[lo:hi] = a @ a2.T
        if train:
            dy = s["dy"][lo:hi].double()
            da = dy @ a2
            if case["act"] == "swiglu":
                dh = torch.cat([da * h[:, I:] * (sig + h[:, :I] * sig * torch.sigmoid(-h[:, :I])), da * h[:, :I] * sig], 1)
            else:
                dh = da * (torch.special.ndtr(h) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi))
            dx[lo:hi], d1[e], d2[e] = dh @ a1, dh.T @ x, dy.T @ a
    return [y, dx, d1, d2] if train else [y]


def _exact_clip(s):
    total = math.sqrt(sum(float(t.double().square().sum()) for t in s["grads"]))
    c = min(1.0, s["max_norm"] / (total + 1e-6))
    return [torch.tensor(total, dtype=torch.float64)] + [t.double() * c for t in s["flat"]]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"gate": _exact_gate, "sort": _exact_sort, "ffn": _exact_ffn, "clip": _exact_clip}[case["op"]](s)
