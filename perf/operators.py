"""What is measured of the operators for language-model training: group norm with an activation (channels last), the
router's top-k gate, tokens sorted by expert and back, and distillation from a teacher's top logits.

A case names its operator (`op`) and its direction (`grad`: with the gradients, from given upstream gradients). `run`
computes the operators in elementary torch operations, or, where `own` is true, with the calls of this repository's C ABI
(`nova_b200.capi`) on the same device buffers.
"""
import math

import torch

own = False

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def listed():
    return [
        # the hidden rows of a small MLP batch at serving time: launch latency
        {"name": "norm rows small", "op": "norm", "batch": 64, "len": 1, "channels": 4096, "groups": 32, "act": "relu", "grad": False},
        # feature maps of 64 x 64 positions with 256 channels, the shape of the reduction benchmark, channels last
        {"name": "norm maps", "op": "norm", "batch": 64, "len": 4096, "channels": 256, "groups": 32, "act": "silu", "grad": False},
        # an odd map (37 x 37) with 10 channels a group, which no 16-byte access divides: a training step's norm
        {"name": "norm odd maps train", "op": "norm", "batch": 16, "len": 1369, "channels": 320, "groups": 32, "act": "silu", "grad": True},
        # the full training batch of the MLP benchmark, 65536 rows of 4096
        {"name": "norm rows train", "op": "norm", "batch": 65536, "len": 1, "channels": 4096, "groups": 32, "act": "gelu", "grad": True},
        # gate of a handful of tokens being decoded
        {"name": "route decode", "op": "route", "tokens": 8, "experts": 64, "k": 2, "renorm": True, "grad": False},
        # gate of a training batch over many experts, weights not renormalised
        {"name": "route train", "op": "route", "tokens": 65536, "experts": 256, "k": 8, "renorm": False, "grad": True},
        # a few tokens sorted by expert, packed
        {"name": "dispatch decode", "op": "dispatch", "tokens": 16, "width": 4096, "experts": 64, "k": 2, "capacity": 0, "grad": False},
        # a training batch into [experts, capacity, width] for the batched product, a quarter of room to spare, and its gradient
        {"name": "dispatch train", "op": "dispatch", "tokens": 16384, "width": 4096, "experts": 64, "k": 4, "capacity": 1280, "grad": True},
        # the way back of the same batch: weighted sums of the experts' rows, and their gradients
        {"name": "combine train", "op": "combine", "tokens": 16384, "width": 4096, "experts": 64, "k": 4, "capacity": 1280, "grad": True},
        # an odd width and an odd number of tokens
        {"name": "combine odd", "op": "combine", "tokens": 1013, "width": 1001, "experts": 7, "k": 2, "capacity": 0, "grad": False},
        # the last positions of a small evaluation batch
        {"name": "distill small", "op": "distill", "rows": 8, "vocab": 32768, "k": 8, "tail": False, "temp": 2.0, "grad": False},
        # a training batch with a large vocabulary, the teacher's mass outside its list in one bucket
        {"name": "distill train", "op": "distill", "rows": 4096, "vocab": 131072, "k": 64, "tail": True, "temp": 1.0, "grad": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "dispatch", "combine", "distill"])
    grad = rng.random() < 0.5
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8, 16, 32, 64])
        channels = groups * _log(rng, 1, 512)
        length = _log(rng, 1, 16384) if rng.random() < 0.7 else 1
        batch = _log(rng, 1, max(1, min(65536, (1 << 27) // (channels * length))))
        # a ReLU's gradient jumps where its argument crosses zero, where no two orders of summation agree
        act = rng.choice(["none", "silu", "gelu"] + ([] if grad else ["relu"]))
        return {"op": op, "batch": batch, "len": length, "channels": channels, "groups": groups, "act": act, "grad": grad}
    if op == "route":
        experts = _log(rng, 2, 512)
        return {"op": op, "tokens": _log(rng, 1, 65536), "experts": experts, "k": rng.randint(1, min(experts, 8)), "renorm": rng.random() < 0.5, "grad": grad}
    if op in ("dispatch", "combine"):
        experts = _log(rng, 1, 256)
        k, tokens = rng.randint(1, min(experts, 8)), _log(rng, 1, 32768)
        width = _log(rng, 1, max(1, min(8192, (1 << 27) // (tokens * k))))
        capacity = rng.choice([0, max(1, math.ceil(1.25 * tokens * k / experts))])
        return {"op": op, "tokens": tokens, "width": width, "experts": experts, "k": k, "capacity": capacity, "grad": grad}
    vocab = _log(rng, 2, 262144)
    rows = _log(rng, 1, max(1, min(8192, (1 << 28) // vocab)))
    return {"op": op, "rows": rows, "vocab": vocab, "k": _log(rng, 1, min(vocab, 256)), "tail": rng.random() < 0.5, "temp": rng.choice([1.0, 2.0, 4.0]), "grad": grad}


def _rows_of(case):
    return case["experts"] * case["capacity"] if case["capacity"] else case["tokens"] * case["k"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "norm":
        shape = (case["batch"], case["len"], case["channels"])
        s["x"] = randn(*shape) * 1.5 + 0.5
        s["gamma"], s["beta"] = 1.0 + 0.2 * randn(case["channels"]), 0.1 * randn(case["channels"])
        s["eps"] = 1e-5
        if case["grad"]:
            s["dy"] = randn(*shape)
    elif case["op"] == "route":
        s["logits"] = randn(case["tokens"], case["experts"]) * 2.0
        if case["grad"]:
            s["dw"] = randn(case["tokens"], case["k"])
    elif case["op"] in ("dispatch", "combine"):
        t, e, k = case["tokens"], case["experts"], case["k"]
        # k distinct experts a token, some experts busier than others; one token in 32 is padding and has none
        liking = randn(1, e) * 0.5 + rand(t, e).log().neg().log().neg()
        ids = liking.argsort(dim=1, descending=True, stable=True)[:, :k].to(torch.int32)
        s["ids"] = torch.where(rand(t, 1) < 1 / 32, torch.full_like(ids, -1), ids).contiguous()
        if case["op"] == "dispatch":
            s["x"] = randn(t, case["width"])
            if case["grad"]:
                s["drows"] = randn(_rows_of(case), case["width"])
        else:
            s["slot"], s["src"], s["counts"] = _sort(s["ids"], e, case["capacity"])
            s["rows_in"] = randn(_rows_of(case), case["width"])
            s["w"] = torch.softmax(randn(t, k), dim=1)
            if case["grad"]:
                s["dout"] = randn(t, case["width"])
    else:
        r, v, k = case["rows"], case["vocab"], case["k"]
        s["z"] = randn(r, v) * 2.0
        # distinct ids a row; the teacher's lists are ordered by logit, not by id
        ids = torch.cumsum(torch.randint(1, max(2, v // k + 1), (r, k), generator=gen, device="cuda"), 1) - 1
        ids = ids[:, torch.randperm(k, generator=gen, device="cuda")]
        # ragged lists: entries past a row's own length are padding; one row in 16 has no teacher at all
        length = torch.randint(1, k + 1, (r, 1), generator=gen, device="cuda")
        length = torch.where(rand(r, 1) < 0.5, torch.full_like(length, k), length)
        length = torch.where(rand(r, 1) < 1 / 16, torch.zeros_like(length), length)
        place = torch.arange(k, device="cuda")[None, :]
        s["ids"] = torch.where(place < length, ids, torch.full_like(ids, -1)).to(torch.int32).contiguous()
        s["t"] = (randn(r, k) * 2.0 + 4.0).sort(dim=1, descending=True).values.contiguous()
        if case["tail"]:
            # the teacher's logsumexp over its whole vocabulary: its list holds between half and nearly all of the mass
            inside = torch.where(s["ids"] >= 0, s["t"] / case["temp"], torch.full_like(s["t"], -1e30)).logsumexp(1)
            s["tlse"] = torch.where(length[:, 0] > 0, inside - torch.log(0.5 + 0.49 * rand(r)), torch.zeros_like(inside))
        if case["grad"]:
            s["dloss"] = (0.5 + rand(r)) / r
    return s


# ---- plain forms


def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _act_slope(v, act):
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "silu":
        sig = 1 / (1 + torch.exp(-v))
        return sig * (1 + v * (1 - sig))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(v)


def _norm(s):
    b, n, c, g = s["batch"], s["len"], s["channels"], s["groups"]
    x = s["x"].view(b, n, g, c // g)
    mean = x.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(dim=(1, 3), keepdim=True) + s["eps"])
    xh = ((x - mean) * rstd).view(b, n, c)
    v = xh * s["gamma"] + s["beta"]
    y = _act(v, s["act"])
    if not s["grad"]:
        return {"y": y}
    dv = s["dy"] * _act_slope(v, s["act"])
    a = (dv * s["gamma"]).view(b, n, g, c // g)
    xg = xh.view(b, n, g, c // g)
    dx = rstd * (a - a.mean(dim=(1, 3), keepdim=True) - xg * (a * xg).mean(dim=(1, 3), keepdim=True))
    return {"y": y, "dx": dx.view(b, n, c), "dgamma": (dv * xh).sum(dim=(0, 1)), "dbeta": dv.sum(dim=(0, 1))}


def _route(s):
    logits, k = s["logits"], s["k"]
    values, order = torch.sort(logits, dim=1, descending=True, stable=True)
    ids, values = order[:, :k], values[:, :k]
    top = values[:, :1]
    below = torch.exp(values - top).sum(1, keepdim=True) if s["renorm"] else torch.exp(logits - top).sum(1, keepdim=True)
    w = torch.exp(values - top) / below
    if not s["grad"]:
        return {"w": w, "ids": ids.to(torch.int32)}
    dot = (w * s["dw"]).sum(1, keepdim=True)
    if s["renorm"]:
        dlogits = torch.zeros_like(logits).scatter(1, ids, w * (s["dw"] - dot))
    else:
        dlogits = (torch.exp(logits - top) / below) * (torch.zeros_like(logits).scatter(1, ids, s["dw"]) - dot)
    return {"w": w, "ids": ids.to(torch.int32), "dlogits": dlogits}


def _sort(ids, experts, capacity):
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=ids.device).scatter_add(0, key, torch.ones_like(key))
    starts = torch.cumsum(counts, 0) - counts
    place = torch.empty_like(key).scatter(0, order, torch.arange(n, device=ids.device) - starts[key[order]])
    keep = key < experts
    if capacity:
        keep = keep & (place < capacity)
    row = (key * capacity if capacity else starts[key]) + place
    rows = experts * capacity if capacity else n
    slot = torch.where(keep, row, torch.full_like(row, -1))
    src = torch.full((rows + 1,), -1, dtype=torch.long, device=ids.device)
    src = src.scatter(0, torch.where(keep, row, torch.full_like(row, rows)), torch.arange(n, device=ids.device))[:rows]
    return slot.view(ids.shape).to(torch.int32), src.to(torch.int32), counts[:experts].to(torch.int32)


def _gather(rows, slot):
    """rows[slot], zeros where there is none."""
    found = rows[slot.clamp(min=0).long()]
    return torch.where((slot >= 0)[..., None], found, torch.zeros_like(found))


def _dispatch(s):
    slot, src, counts = _sort(s["ids"], s["experts"], s["capacity"])
    token = torch.div(src.clamp(min=0), s["k"], rounding_mode="floor").long()
    rows = torch.where((src >= 0)[:, None], s["x"][token], torch.zeros((), device=src.device))
    out = {"slot": slot, "src": src, "counts": counts, "rows": rows}
    if s["grad"]:
        out["dx"] = _gather(s["drows"], slot).sum(1)
    return out


def _combine(s):
    slot, src, w = s["slot"], s["src"], s["w"]
    found = _gather(s["rows_in"], slot)
    out = {"out": (w[:, :, None] * found).sum(1)}
    if s["grad"]:
        out["dw"] = (s["dout"][:, None, :] * found).sum(2)
        at = src.clamp(min=0).long()
        token = torch.div(at, s["k"], rounding_mode="floor")
        out["drows"] = torch.where((src >= 0)[:, None], w.reshape(-1)[at][:, None] * s["dout"][token], torch.zeros((), device=src.device))
    return out


def _distill(s):
    z, ids, tau = s["z"], s["ids"], s["temp"]
    valid = ids >= 0
    some = valid.any(1)
    at = ids.clamp(min=0).long()
    top = z.max(1, keepdim=True).values
    lse = torch.log(torch.exp((z - top) / tau).sum(1, keepdim=True)) + top / tau
    t = torch.where(valid, s["t"] / tau, torch.full_like(s["t"], -math.inf))
    if s["tail"]:
        logp = t - s["tlse"][:, None]
    else:
        t_top = torch.where(some[:, None], t.max(1, keepdim=True).values, torch.zeros_like(lse))
        total = torch.exp(t - t_top).sum(1, keepdim=True)
        logp = t - t_top - torch.log(torch.where(some[:, None], total, torch.ones_like(total)))
    p = torch.exp(logp)
    logq = torch.gather(z, 1, at) / tau - lse
    zero = torch.zeros_like(p)
    loss = torch.where(p > 0, p * (torch.where(p > 0, logp, zero) - logq), zero).sum(1)
    mass = p.sum(1)
    if s["tail"]:
        # a row's list, marked in the vocabulary (padding marks a column behind it)
        inside = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.bool, device=z.device)
        inside = inside.scatter(1, torch.where(valid, at, torch.full_like(at, z.shape[1])), True)[:, :-1]
        outside = z.masked_fill(inside, -math.inf)
        o_top = outside.max(1, keepdim=True).values
        o_top = torch.where(torch.isinf(o_top), top, o_top)
        tail_lse = torch.log(torch.exp((outside - o_top) / tau).sum(1, keepdim=True)) + o_top / tau
        p_tail = (1 - mass).clamp(min=0)
        some_tail = p_tail > 0
        term = p_tail * (torch.log(torch.where(some_tail, p_tail, torch.ones_like(p_tail))) - (tail_lse - lse)[:, 0])
        loss = loss + torch.where(some_tail, term, torch.zeros_like(term))
        mass = mass + p_tail
    out = {"loss": torch.where(some, tau * tau * loss, torch.zeros_like(loss))}
    if s["grad"]:
        dz = mass[:, None] * torch.exp(z / tau - lse)
        if s["tail"]:
            dz = dz - torch.where(some_tail[:, None], p_tail[:, None] * torch.exp(outside / tau - tail_lse).masked_fill(inside, 0.0), torch.zeros_like(lse))
        dz = dz.scatter_add(1, at, torch.where(valid, -p, zero))
        out["dz"] = torch.where(some[:, None], (tau * s["dloss"])[:, None] * dz, torch.zeros_like(lse))
    return out


# ---- the framework's calls


def _own(s):
    from nova_b200 import capi

    lib = capi.lib()
    # a null stream is the library's own; torch's default stream goes by the handle of the legacy default stream
    stream = torch.cuda.current_stream().cuda_stream or 1
    new = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    new_ids = lambda *shape: torch.empty(shape, device="cuda", dtype=torch.int32)  # noqa: E731
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if s["op"] == "norm":
        x, act = s["x"], ACTS[s["act"]]
        b, n, c, g = s["batch"], s["len"], s["channels"], s["groups"]
        y, stats = torch.empty_like(x), new(2, b, g)
        size = capi.group_norm_workspace(b, n, c, g, s["grad"])
        work = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
        capi.check(lib.fz_group_norm(at(y), at(stats[0]), at(stats[1]), at(x), at(s["gamma"]), at(s["beta"]), b, n, c, g, s["eps"], act, at(work), size, stream))
        if not s["grad"]:
            return {"y": y}
        dx, dgb = torch.empty_like(x), new(2, c)
        capi.check(lib.fz_group_norm_backward(at(dx), at(dgb[0]), at(dgb[1]), at(s["dy"]), at(x), at(stats[0]), at(stats[1]), at(s["gamma"]), at(s["beta"]),
                                              b, n, c, g, act, at(work), size, stream))
        return {"y": y, "dx": dx, "dgamma": dgb[0], "dbeta": dgb[1]}
    if s["op"] == "route":
        t, e, k = s["tokens"], s["experts"], s["k"]
        w, ids = new(t, k), new_ids(t, k)
        capi.check(lib.fz_route(at(w), at(ids), at(s["logits"]), t, e, k, s["renorm"], stream))
        if not s["grad"]:
            return {"w": w, "ids": ids}
        dlogits = new(t, e)
        capi.check(lib.fz_route_backward(at(dlogits), at(s["dw"]), at(w), at(ids), at(s["logits"]), t, e, k, s["renorm"], stream))
        return {"w": w, "ids": ids, "dlogits": dlogits}
    if s["op"] == "dispatch":
        t, d, e, k, r = s["tokens"], s["width"], s["experts"], s["k"], _rows_of(s)
        slot, src, counts, offsets, rows = new_ids(t, k), new_ids(r), new_ids(e), new_ids(e + 1), new(r, d)
        capi.check(lib.fz_expert_sort(at(slot), at(src), at(counts), at(offsets), at(s["ids"]), t, k, e, s["capacity"], stream))
        capi.check(lib.fz_expert_dispatch(at(rows), at(s["x"]), at(slot), at(src), t, k, r, d, stream))
        out = {"slot": slot, "src": src, "counts": counts, "rows": rows}
        if s["grad"]:
            out["dx"] = new(t, d)
            capi.check(lib.fz_expert_combine(at(out["dx"]), at(s["drows"]), None, at(slot), t, k, r, d, stream))
        return out
    if s["op"] == "combine":
        t, d, k, r = s["tokens"], s["width"], s["k"], _rows_of(s)
        out = {"out": new(t, d)}
        capi.check(lib.fz_expert_combine(at(out["out"]), at(s["rows_in"]), at(s["w"]), at(s["slot"]), t, k, r, d, stream))
        if s["grad"]:
            out["dw"], out["drows"] = new(t, k), new(r, d)
            capi.check(lib.fz_expert_combine_backward(at(out["drows"]), at(out["dw"]), at(s["dout"]), at(s["rows_in"]), at(s["w"]), at(s["slot"]), at(s["src"]), t, k, r, d, stream))
        return out
    z, r, v, k, tlse = s["z"], s["rows"], s["vocab"], s["k"], s.get("tlse")
    loss, stats = new(r), new(r, 4)
    capi.check(lib.fz_distill(at(loss), at(stats), at(z), v, at(s["ids"]), at(s["t"]), at(tlse), r, v, k, s["temp"], stream))
    if not s["grad"]:
        return {"loss": loss}
    dz = torch.empty_like(z)
    capi.check(lib.fz_distill_backward(at(dz), v, at(s["dloss"]), at(stats), at(z), v, at(s["ids"]), at(s["t"]), at(tlse), r, v, k, s["temp"], stream))
    return {"loss": loss, "dz": dz}


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "route": _route, "dispatch": _dispatch, "combine": _combine, "distill": _distill}[state["op"]](state)


def work(case):
    op, grad = case["op"], case["grad"]
    if op == "norm":
        n = case["batch"] * case["len"] * case["channels"]
        return {"bytes": 4 * n * (5 if grad else 2), "flops": n * (30 if grad else 10)}
    if op == "route":
        n, picks = case["tokens"] * case["experts"], case["tokens"] * case["k"]
        moved = n + 2 * picks
        if grad:
            moved += picks + n * (1 if case["renorm"] else 2)
        return {"bytes": 4 * moved, "flops": n * (case["k"] + 2)}
    if op in ("dispatch", "combine"):
        t, d, picks, rows = case["tokens"], case["width"], case["tokens"] * case["k"], _rows_of(case)
        filled = min(picks, rows)
        if op == "dispatch":
            moved = 2 * picks + rows + t * d + rows * d + (filled * d + t * d if grad else 0)
            return {"bytes": 4 * moved, "flops": picks * d if grad else picks}
        moved = 2 * picks + filled * d + t * d + (t * d + rows * d + filled * d + picks if grad else 0)
        return {"bytes": 4 * moved, "flops": picks * d * (5 if grad else 2)}
    n, picks = case["rows"] * case["vocab"], case["rows"] * case["k"]
    return {"bytes": 4 * (n * (3 if grad else 1) + 2 * picks + case["rows"]), "flops": n * (8 if grad else 4)}


# ---- from the definitions, in 64 bits


def _exact_norm(s):
    b, n, c, g = s["batch"], s["len"], s["channels"], s["groups"]
    x = s["x"].double().reshape(b, n, g, c // g).transpose(1, 2).reshape(b * g, -1)
    mean = x.sum(1, keepdim=True) / x.shape[1]
    x = x - mean
    sigma = torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + s["eps"])
    back = lambda u: u.reshape(b, g, n, c // g).transpose(1, 2).reshape(b, n, c)  # noqa: E731
    x = back(x / sigma)
    v = torch.addcmul(s["beta"].double(), x, s["gamma"].double())
    phi = lambda u: torch.special.ndtr(u)  # noqa: E731
    y = {"none": lambda: v, "relu": lambda: v.clamp(min=0), "silu": lambda: v * torch.sigmoid(v), "gelu": lambda: v * phi(v)}[s["act"]]()
    if not s["grad"]:
        return {"y": y}
    slope = {"none": lambda: torch.ones_like(v), "relu": lambda: torch.sign(v).clamp(min=0), "silu": lambda: torch.sigmoid(v) + y * torch.sigmoid(-v),
             "gelu": lambda: phi(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)}[s["act"]]()
    dv = slope * s["dy"].double()
    del slope, v
    flat = lambda u: u.reshape(b, n, g, c // g).transpose(1, 2).reshape(b * g, -1)  # noqa: E731
    a, xg = flat(dv * s["gamma"].double()), flat(x)
    m = a.shape[1]
    # the gradient through (x - mean) / sigma: off the span of the ones and of xh
    dx = (a - a.sum(1, keepdim=True) / m - xg * ((a * xg).sum(1, keepdim=True) / m)) / sigma
    return {"y": y, "dx": back(dx), "dgamma": torch.einsum("blc,blc->c", dv, x), "dbeta": dv.sum((0, 1))}


def _exact_route(s):
    logits = s["logits"].double()
    picked = torch.argsort(-logits, dim=1, stable=True)[:, : s["k"]]
    chosen = torch.zeros_like(logits).scatter(1, picked, 1.0)
    over = torch.where(chosen > 0, logits, torch.full_like(logits, -math.inf)) if s["renorm"] else logits
    p = torch.softmax(over, 1)
    out = {"w": p.gather(1, picked), "ids": None}
    if s["grad"]:
        up = torch.zeros_like(p).scatter(1, picked, s["dw"].double())
        out["dlogits"] = p * up - p * (p * up).sum(1, keepdim=True)
    return out


def _exact_dispatch(s):
    _, src, _ = _sort(s["ids"], s["experts"], s["capacity"])
    held = src >= 0
    rows = torch.zeros((src.numel(), s["width"]), dtype=torch.float64, device=src.device)
    rows[held] = s["x"].double()[src[held].long() // s["k"]]
    out = {"slot": None, "src": None, "counts": None, "rows": rows}
    if s["grad"]:
        dx = torch.zeros((s["tokens"], s["width"]), dtype=torch.float64, device=src.device)
        out["dx"] = dx.index_add(0, src[held].long() // s["k"], s["drows"].double()[held])
    return out


def _exact_combine(s):
    held = s["src"] >= 0
    at = s["src"][held].long()
    token = at // s["k"]
    weight, rows = s["w"].double().reshape(-1)[at], s["rows_in"].double()[held]
    zeros = lambda *n: torch.zeros(n, dtype=torch.float64, device=at.device)  # noqa: E731
    out = {"out": zeros(s["tokens"], s["width"]).index_add(0, token, rows * weight[:, None])}
    if s["grad"]:
        dout = s["dout"].double()[token]
        out["dw"] = zeros(s["w"].numel()).index_copy(0, at, torch.einsum("rd,rd->r", dout, rows)).view(s["w"].shape)
        out["drows"] = zeros(held.numel(), s["width"])
        out["drows"][held] = dout * weight[:, None]
    return out


def _exact_distill(s):
    tau, ids = s["temp"], s["ids"]
    z, valid = s["z"].double() / tau, ids >= 0
    some, v = valid.any(1), z.shape[1]
    logq = torch.log_softmax(z, 1)
    # the teacher spread over the vocabulary, one column more for padding
    column = torch.where(valid, ids.long(), torch.full_like(ids, v, dtype=torch.long))
    spread = torch.full((z.shape[0], v + 1), -math.inf, dtype=torch.float64, device=z.device)
    spread = spread.scatter(1, column, s["t"].double() / tau)[:, :v]
    logp = spread - (s["tlse"].double()[:, None] if s["tail"] else torch.logsumexp(spread, 1, keepdim=True))
    logp = torch.where(some[:, None], logp, torch.full_like(logp, -math.inf))
    p = torch.exp(logp)
    loss = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
    del logp
    q = torch.exp(logq)
    dz = p.sum(1, keepdim=True) * q - p
    if s["tail"]:
        rest = (1 - p.sum(1)).clamp(min=0)
        outside = torch.where(torch.isinf(spread), logq, torch.full_like(logq, -math.inf))
        log_rest = torch.logsumexp(outside, 1)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_rest), torch.zeros_like(rest))
        dz = dz + rest[:, None] * (q - torch.where((rest > 0)[:, None] & torch.isinf(spread), torch.exp(outside - log_rest[:, None]), torch.zeros_like(q)))
    zero = torch.zeros((), dtype=torch.float64, device=z.device)
    out = {"loss": torch.where(some, tau * tau * loss, zero)}
    if s["grad"]:
        out["dz"] = torch.where(some[:, None], dz * (tau * s["dloss"].double())[:, None], zero)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "dispatch": _exact_dispatch, "combine": _exact_combine, "distill": _exact_distill}[case["op"]](s)
