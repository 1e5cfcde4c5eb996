"""The bf16 expert layer in its parts, as cases that can be timed: tokens sorted by expert and back with their
weights, matrix products with their epilogue (dense, or one matrix per expert over the sorted rows), and the
gradients of both.

  dispatch      ops.moe_sort + ops.moe_gather: (token, slot) pairs in the order of their experts, the tokens' rows
                copied to that order; ids that are no expert here (-1: an expert of another GPU) are dropped
  combine       ops.moe_combine: every token's rows summed with its weights, plus a residual
  combine_grad  ops.moe_combine_grad: the gradient of the rows and of the weights
  linear        ops.linear: act(x w^T + bias) + residual
  experts       ops.linear with an order: row p through the matrix of the expert that it is sorted under
  linear_grad   ops.linear_grad: the gradient of x, w and bias; experts_grad: the same with an order
act is None, "silu" or "swiglu" (silu(min(g, L)) * clamp(u, -L, L) of two products g and u, as the framework's
experts have it).  Sizes are those of MoEConfig (hidden 4096, expert 2048, 256 experts, top 6) and, among the drawn
ones, generic ones.
"""
import math

import torch

own = False  # True: the framework's operators, False: their plain form

DEVICE = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
LIMIT = 10.0
SCALING = 1.5


def listed():
    return [
        # plain decode of one token: what is left is latency
        {"name": "dispatch_1", "kind": "dispatch", "m": 1, "k": 6, "experts": 256, "d": 4096, "type": "bf16",
         "zipf": 0.0, "drop": 0.0},
        # a long prompt with a skewed popularity of the experts, a quarter of which live on another GPU
        {"name": "dispatch_4096", "kind": "dispatch", "m": 4096, "k": 6, "experts": 256, "d": 4096, "type": "bf16",
         "zipf": 1.1, "drop": 0.25},
        # a verify's token and its drafts, from fp32 rows
        {"name": "combine_5", "kind": "combine", "m": 5, "k": 6, "experts": 256, "d": 4096, "type": "f32", "out": "bf16",
         "residual": True, "zipf": 0.0, "drop": 0.0},
        # a long prompt, the shared expert's rows as the residual
        {"name": "combine_4096", "kind": "combine", "m": 4096, "k": 6, "experts": 256, "d": 4096, "type": "bf16",
         "out": "bf16", "residual": True, "zipf": 1.1, "drop": 0.0},
        # the way back of a training step, the weights' gradient on its way to the router
        {"name": "combine_grad_4096", "kind": "combine_grad", "m": 4096, "k": 6, "experts": 64, "d": 4096,
         "type": "bf16", "out": "bf16", "residual": False, "zipf": 0.5, "drop": 0.0},
        # a projection of one token added to another one's result (the draft block's input): the weights' stream
        {"name": "linear_1", "kind": "linear", "m": 1, "n": 4096, "kk": 4096, "act": "none", "bias": False,
         "residual": True, "pre": False, "out": "bf16"},
        # the gate and up products of a shared expert over a ragged prompt: few tiles
        {"name": "linear_500", "kind": "linear", "m": 500, "n": 2048, "kk": 4096, "act": "swiglu", "bias": False,
         "residual": False, "pre": False, "out": "bf16"},
        # a square projection of a long ragged prompt, everything in the epilogue
        {"name": "linear_4093", "kind": "linear", "m": 4093, "n": 4096, "kk": 4096, "act": "silu", "bias": True,
         "residual": True, "pre": False, "out": "bf16"},
        # eight sequences decoding together: one or two rows per expert, the weights' stream
        {"name": "experts_8", "kind": "experts", "m": 8, "k": 6, "experts": 256, "n": 2048, "kk": 4096, "act": "swiglu",
         "bias": False, "residual": False, "pre": False, "out": "bf16", "zipf": 0.0, "drop": 0.0},
        # the forward pass of a training step: gate and up of all experts, kept for the backward pass
        {"name": "experts_2048", "kind": "experts", "m": 2048, "k": 6, "experts": 64, "n": 2048, "kk": 4096,
         "act": "swiglu", "bias": False, "residual": False, "pre": True, "out": "bf16", "zipf": 0.5, "drop": 0.0},
        # a dense layer's backward pass over a ragged batch
        {"name": "linear_grad_1001", "kind": "linear_grad", "m": 1001, "n": 4096, "kk": 4096, "act": "none",
         "bias": True},
        # the backward pass of the experts' gate and up
        {"name": "experts_grad_2048", "kind": "experts_grad", "m": 2048, "k": 6, "experts": 64, "n": 2048, "kk": 4096,
         "act": "swiglu", "bias": False, "zipf": 0.5, "drop": 0.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _times8(rng, lo, hi):
    return 8 * _log_int(rng, lo // 8, hi // 8)


def draw(rng):
    kind = rng.choice(("dispatch", "combine", "combine_grad", "linear", "linear", "experts", "experts", "linear_grad",
                       "experts_grad"))
    case = {"kind": kind, "m": _log_int(rng, 1, 4096)}
    if kind not in ("linear", "linear_grad"):
        case.update(experts=_log_int(rng, 2, 256), zipf=round(rng.uniform(0.0, 1.3), 2),
                    drop=rng.choice((0.0, 0.0, round(rng.uniform(0.0, 1.0), 2))))
        case["k"] = rng.randint(1, min(8, case["experts"]))
    if kind in ("dispatch", "combine", "combine_grad"):
        case.update(d=rng.choice((_times8(rng, 64, 4096), _times8(rng, 64, 4096), _log_int(rng, 64, 4096), 4096)),
                    type=rng.choice(("bf16", "bf16", "f32")))
        if kind != "dispatch":
            case.update(out=rng.choice(("bf16", "bf16", "f32")), residual=rng.random() < 0.5)
        return case
    case.update(n=_times8(rng, 64, 4096), kk=_times8(rng, 64, 4096), act=rng.choice(("none", "silu", "swiglu")),
                bias=rng.random() < 0.5)
    if kind in ("linear", "experts"):
        case.update(residual=rng.random() < 0.5, pre=rng.random() < 0.3, out=rng.choice(("bf16", "bf16", "f32")))
    if kind.startswith("experts"):
        case["m"] = _log_int(rng, 1, 2048)
        # no more than the largest listed case's matrices and products
        mats = 2 if case["act"] == "swiglu" else 1
        case["experts"] = max(case["k"], min(case["experts"], (1 << 30) // (mats * case["n"] * case["kk"])))
        while work(case)["flops"] > (8e11 if kind == "experts_grad" else 4e11):
            case["m"] = (case["m"] + 1) // 2
    return case


# ---------------------------------------------------------------- inputs

def _gen(seed, sub):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 64 + sub)
    return g


def _normal(seed, sub, shape, std, dtype=BF16):
    return torch.randn(shape, generator=_gen(seed, sub), device=DEVICE, dtype=dtype).mul_(std)


def _dtype(name):
    return F32 if name == "f32" else BF16


def _routing(case, seed):
    """ids int64 [m, k], distinct in a token, popularity falling as 1 / rank^zipf; weights fp32 that sum to SCALING."""
    e, m, k = case["experts"], case["m"], case["k"]
    u = torch.rand((m, e), generator=_gen(seed, 1), device=DEVICE).clamp_(1e-20)
    logp = -case["zipf"] * torch.arange(1, e + 1, device=DEVICE, dtype=F32).log()
    idx = (logp - (-u.log()).clamp_(min=1e-20).log()).topk(k, dim=1).indices
    popular = torch.randperm(e, generator=_gen(seed, 2), device=DEVICE)
    idx = popular[idx]
    if case["drop"]:  # the experts of other GPUs
        away = torch.rand(e, generator=_gen(seed, 3), device=DEVICE) < case["drop"]
        idx = torch.where(away[idx], -1, idx)
    w = torch.rand((m, k), generator=_gen(seed, 4), device=DEVICE) + 0.1
    return idx, w / w.sum(dim=1, keepdim=True) * SCALING


def _order(idx, experts):
    """offsets int32 [E + 1], the pair of each row int32 [M k] (-1 behind the last), the row of each pair [M, k]."""
    flat = idx.reshape(-1)
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, experts)
    perm = torch.sort(key, stable=True).indices
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((counts.new_zeros(1), counts[:experts].cumsum(0)))
    pairs = torch.where(valid[perm], perm, -1)
    rows = torch.empty_like(flat).scatter_(0, perm, torch.arange(flat.numel(), device=flat.device))
    rows = torch.where(valid, rows, -1)
    return offsets.to(torch.int32), pairs.to(torch.int32), rows.to(torch.int32).reshape(idx.shape)


def prepare(case, seed):
    """Inputs from the seed, weights, and the order of the rows where the pass starts from sorted ones."""
    kind, m = case["kind"], case["m"]
    state = {"kind": kind, "case": case}
    sorted_rows = kind not in ("linear", "linear_grad")
    if sorted_rows:
        state["idx"], state["w"] = _routing(case, seed)
        if kind != "dispatch":
            state["order"] = _order(state["idx"], case["experts"])
    if kind == "dispatch":
        state["x"] = _normal(seed, 5, (m, case["d"]), 1.0, _dtype(case["type"]))
        return state
    if kind in ("combine", "combine_grad"):
        state["rows"] = _normal(seed, 5, (m * case["k"], case["d"]), 1.0, _dtype(case["type"]))
        if kind == "combine_grad":
            state["d_out"] = _normal(seed, 6, (m, case["d"]), 1.0, _dtype(case["out"]))
        elif case["residual"]:
            state["residual"] = _normal(seed, 6, (m, case["d"]), 1.0, _dtype(case["out"]))
        return state
    p, n, kk = (m * case["k"] if sorted_rows else m), case["n"], case["kk"]
    lead = (case["experts"],) if sorted_rows else ()
    names = ("w", "w_up") if case["act"] == "swiglu" else ("w",)
    state["x"] = _normal(seed, 5, (p, kk), 1.0)
    for j, name in enumerate(names):  # products of unit size, some of them beyond the limit of swiglu
        state[name] = _normal(seed, 7 + j, lead + (n, kk), (3.0 if case["act"] == "swiglu" else 1.0) / math.sqrt(kk))
        if case["bias"] and kind in ("linear", "experts"):
            state["bias" + name[1:]] = _normal(seed, 9 + j, lead + (n,), 0.5)
    if kind in ("linear", "experts"):
        if case["residual"]:
            state["residual"] = _normal(seed, 6, (p, n), 1.0)
    else:
        state["d_out"] = _normal(seed, 11, (p, n), 1.0)
        if case["act"] != "none":  # what the forward pass kept: x w^T + bias, gate and up side by side
            state["pre"] = _normal(seed, 12, (p, n * len(names)), 3.0)
    return state


# ---------------------------------------------------------------- the pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import __graft_entry__
    __graft_entry__.package()
    from home_seek_amd import ops

    kind, case = state["kind"], state["case"]
    if kind == "dispatch":
        order = ops.moe_sort(state["idx"], case["experts"])
        rows = ops.moe_gather(state["x"], order)
        return {"offsets": order.offsets, "pairs": order.pairs, "rows_of": order.rows, "rows": rows}
    order = ops.ExpertOrder(*state["order"]) if "order" in state else None
    if kind == "combine":
        return ops.moe_combine(state["rows"], order, state["w"], state.get("residual"), out_dtype=_dtype(case["out"]))
    if kind == "combine_grad":
        d_rows, d_w = ops.moe_combine_grad(state["d_out"], state["rows"], order, state["w"])
        return {"d_rows": d_rows, "d_w": d_w}
    act = None if case["act"] == "none" else case["act"]
    limit = LIMIT if act == "swiglu" else None
    if kind in ("linear", "experts"):
        return ops.linear(state["x"], state["w"], state.get("bias"), state.get("residual"), act=act,
                          w_up=state.get("w_up"), bias_up=state.get("bias_up"), limit=limit, order=order,
                          out_dtype=_dtype(case["out"]), want_pre=case["pre"])
    g = ops.linear_grad(state["d_out"], state["x"], state["w"], act=act, pre=state.get("pre"), w_up=state.get("w_up"),
                        limit=limit, order=order, need_bias=case["bias"])
    return [t for t in g if t is not None]


def _act_plain(act, z, z_up):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "swiglu":
        g, u = z.clamp(max=LIMIT), z_up.clamp(-LIMIT, LIMIT)
        return g * torch.sigmoid(g) * u
    return z


def _groups(state):
    """(expert, first row, end) of what has rows; a dense product is one group."""
    if "order" not in state:
        return [(None, 0, state["x"].shape[0])]
    off = state["order"][0].tolist()
    return [(e, a, b) for e, (a, b) in enumerate(zip(off[:-1], off[1:])) if b > a]


def _of(t, e):
    return None if t is None else (t if e is None else t[e]).float()


def _run_plain(state):
    kind, case = state["kind"], state["case"]
    if kind == "dispatch":
        k = case["k"]
        offsets, pairs, rows_of = _order(state["idx"], case["experts"])
        rows = state["x"][(pairs.clamp(min=0) // k).long()] * (pairs >= 0)[:, None]
        return {"offsets": offsets, "pairs": pairs, "rows_of": rows_of, "rows": rows}
    if kind == "combine":
        rows_of = state["order"][2]
        picked = state["rows"][rows_of.clamp(min=0).long()].float()
        picked = torch.where((rows_of >= 0)[:, :, None], picked * state["w"][:, :, None], 0.0)
        out = picked.sum(dim=1)
        if "residual" in state:
            out = out + state["residual"].float()
        return out.to(_dtype(case["out"]))
    if kind == "combine_grad":
        _, pairs, rows_of = state["order"]
        k = case["k"]
        p = pairs.clamp(min=0).long()
        per_row = state["d_out"].float()[p // k]
        d_rows = torch.where((pairs >= 0)[:, None], per_row * state["w"].reshape(-1)[p][:, None], 0.0)
        dots = (per_row * state["rows"].float()).sum(dim=1)
        d_w = torch.where(rows_of >= 0, dots[rows_of.clamp(min=0).long()], 0.0)
        return {"d_rows": d_rows.to(state["rows"].dtype), "d_w": d_w}
    act, x, n = case["act"], state["x"], case["n"]
    if kind in ("linear", "experts"):
        out = torch.zeros(x.shape[0], n, dtype=F32, device=x.device)
        pre = torch.zeros(x.shape[0], n * (2 if act == "swiglu" else 1), dtype=F32, device=x.device)
        for e, a, b in _groups(state):
            zs = []
            for name in ("w", "w_up")[: 2 if act == "swiglu" else 1]:
                z = x[a:b].float() @ _of(state[name], e).T
                if "bias" + name[1:] in state:
                    z = z + _of(state["bias" + name[1:]], e)
                zs.append(z)
            out[a:b] = _act_plain(act, *(zs + [None])[:2])
            if "residual" in state:
                out[a:b] += state["residual"][a:b].float()
            if case["pre"]:
                pre[a:b] = torch.cat(zs, dim=1)
        out = out.to(_dtype(case["out"]))
        return (out, pre.to(BF16)) if case["pre"] else out
    d_out = state["d_out"].float()
    if act == "none":
        dz = [d_out]
    else:
        z = state["pre"].float()
        g = z[:, :n].clamp(max=LIMIT) if act == "swiglu" else z
        s = torch.sigmoid(g)
        dz = [d_out * (s + g * s * (1 - s))]
        if act == "swiglu":
            u = z[:, n:].clamp(-LIMIT, LIMIT)
            dz = [torch.where(z[:, :n] <= LIMIT, dz[0] * u, 0.0),
                  torch.where(z[:, n:].abs() <= LIMIT, d_out * g * s, 0.0)]
    names = ("w", "w_up")[: len(dz)]
    dx = torch.zeros(x.shape, dtype=F32, device=x.device)
    dw = [torch.zeros(state[name].shape, dtype=BF16, device=x.device) for name in names]
    db = [torch.zeros(state[name].shape[:-1], dtype=F32, device=x.device) for name in names]
    for e, a, b in _groups(state):
        for j, name in enumerate(names):
            dx[a:b] += dz[j][a:b] @ _of(state[name], e)
            (dw[j] if e is None else dw[j][e]).copy_(dz[j][a:b].T @ x[a:b].float())
            (db[j] if e is None else db[j][e]).copy_(dz[j][a:b].sum(dim=0))
    outs = [dx.to(BF16), dw[0]] + ([db[0]] if case["bias"] else [])
    if act == "swiglu":
        outs += [dw[1]] + ([db[1]] if case["bias"] else [])
    return outs


# ---------------------------------------------------------------- what a pass cannot do without

def _live(case):
    """Rows that are sorted under an expert, and experts that have any, on average."""
    e, m, k = case["experts"], case["m"], case["k"]
    p = torch.arange(1, e + 1, dtype=torch.float64) ** -case["zipf"]
    share = (p / p.sum() * k).clamp(max=1.0)
    keep = 1.0 - case["drop"]
    return m * k * keep, float((1.0 - (1.0 - share) ** m).sum()) * keep


def work(case):
    kind, m = case["kind"], case["m"]
    size = {"bf16": 2, "f32": 4}
    if kind in ("dispatch", "combine", "combine_grad"):
        k, d, s = case["k"], case["d"], size[case["type"]]
        live, _ = _live(case)
        pairs = m * k
        if kind == "dispatch":  # ids; the tokens; all rows, those behind the last as zeros; the order
            return {"bytes": float(8 * pairs + m * d * s + pairs * d * s + 8 * pairs + 4 * case["experts"]), "flops": 0.0}
        o = size[case["out"]]
        if kind == "combine":
            nbytes = live * d * s + 8 * pairs + m * d * o * (2 if case["residual"] else 1)
            return {"bytes": float(nbytes), "flops": 2.0 * live * d}
        return {"bytes": float(live * d * s + pairs * d * s + m * d * o + 16 * pairs), "flops": 3.0 * live * d}
    n, kk, mats = case["n"], case["kk"], 2 if case["act"] == "swiglu" else 1
    if kind.startswith("experts"):
        live, touched = _live(case)
        total, every = m * case["k"], case["experts"]
    else:
        live, touched, total, every = m, 1, m, 1
    flops = 2.0 * live * n * kk * mats
    if kind in ("linear", "experts"):
        o = size[case["out"]]
        nbytes = 2 * live * kk + 2 * touched * n * kk * mats + total * n * o + (2 * live * n if case["residual"] else 0)
        nbytes += 2 * total * n * mats if case["pre"] else 0
        return {"bytes": float(nbytes), "flops": flops}
    nbytes = 2 * live * n * (1 + (mats if case["act"] != "none" else 0)) + 2 * live * kk + 2 * total * kk
    nbytes += 2 * touched * n * kk * mats + 2 * every * n * kk * mats
    return {"bytes": float(nbytes), "flops": 2.0 * flops}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """From the definitions, token by token and expert by expert, in 64 bits."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "dispatch":
        rows = torch.zeros(case["m"] * case["k"], case["d"], dtype=torch.float64, device=DEVICE)
        at = 0
        for e in range(case["experts"]):
            token = torch.nonzero(state["idx"] == e)[:, 0]  # in the order of the pairs
            rows[at:at + len(token)] = state["x"][token].double()
            at += len(token)
        return {"offsets": None, "pairs": None, "rows_of": None, "rows": rows}
    if kind == "combine":
        rows_of, w = state["order"][2], state["w"].double()
        out = torch.zeros(case["m"], case["d"], dtype=torch.float64, device=DEVICE)
        for j in range(case["k"]):
            t = torch.nonzero(rows_of[:, j] >= 0)[:, 0]
            out[t] += w[t, j, None] * state["rows"][rows_of[t, j].long()].double()
        return out + state["residual"].double() if case["residual"] else out
    if kind == "combine_grad":
        rows_of, w, d_out = state["order"][2], state["w"].double(), state["d_out"].double()
        d_rows = torch.zeros(state["rows"].shape, dtype=torch.float64, device=DEVICE)
        d_w = torch.zeros(w.shape, dtype=torch.float64, device=DEVICE)
        for j in range(case["k"]):
            t = torch.nonzero(rows_of[:, j] >= 0)[:, 0]
            r = rows_of[t, j].long()
            d_rows[r] = w[t, j, None] * d_out[t]
            d_w[t, j] = (d_out[t] * state["rows"][r].double()).sum(dim=1)
        return {"d_rows": d_rows, "d_w": d_w}
    x, act = state["x"].double(), case["act"]
    pairs = 2 if act == "swiglu" else 1
    spans = [(0, x.shape[0])]
    if "order" in state:
        off = state["order"][0].tolist()
        spans = list(zip(off[:-1], off[1:]))

    def mat(name, g):
        return (state[name][g] if "order" in state else state[name]).double()

    if kind in ("linear", "experts"):
        out = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=DEVICE)
        pre = torch.zeros(x.shape[0], case["n"] * pairs, dtype=torch.float64, device=DEVICE)
        for g, (a, b) in enumerate(spans):
            if a == b:
                continue
            z = torch.matmul(x[a:b], mat("w", g).t())
            z = z + mat("bias", g) if "bias" in state else z
            y = z
            if act == "silu":
                y = z / (1 + torch.exp(-z))
            if act == "swiglu":
                zu = torch.matmul(x[a:b], mat("w_up", g).t())
                zu = zu + mat("bias_up", g) if "bias_up" in state else zu
                gate = torch.minimum(z, z.new_tensor(LIMIT))
                up = torch.maximum(torch.minimum(zu, z.new_tensor(LIMIT)), z.new_tensor(-LIMIT))
                y = gate / (1 + torch.exp(-gate)) * up
                z = torch.cat((z, zu), dim=1)
            out[a:b] = y + state["residual"][a:b].double() if case["residual"] else y
            pre[a:b] = z
        return (out, pre) if case["pre"] else out
    n, d = case["n"], state["d_out"].double()
    if act == "none":
        dz = d
    else:
        z = state["pre"].double()
        gate = torch.minimum(z[:, :n], z.new_tensor(LIMIT)) if act == "swiglu" else z
        sig = 1 / (1 + torch.exp(-gate))
        slope = sig * (1 + gate * (1 - sig))
        if act == "silu":
            dz = d * slope
        else:
            zu = z[:, n:]
            up = torch.maximum(torch.minimum(zu, z.new_tensor(LIMIT)), z.new_tensor(-LIMIT))
            dz = torch.cat((d * up * slope * (z[:, :n] <= LIMIT), d * gate * sig * (zu >= -LIMIT) * (zu <= LIMIT)), dim=1)
    dx = torch.zeros_like(x)
    shape = state["w"].shape
    dw = [torch.zeros(shape, dtype=F32, device=DEVICE) for _ in range(pairs)]  # held in 32 bits: an error of 2^-24
    db = [torch.zeros(shape[:-1], dtype=torch.float64, device=DEVICE) for _ in range(pairs)]
    for g, (a, b) in enumerate(spans):
        for j in range(pairs):
            part = dz[a:b, j * n:(j + 1) * n]
            dx[a:b] += torch.matmul(part, mat("w_up" if j else "w", g))
            at = (g,) if "order" in state else (slice(None),)
            dw[j][at] = torch.matmul(part.t(), x[a:b]).float()
            db[j][at] = part.sum(dim=0)
    outs = [dx]
    for j in range(pairs):
        outs += [dw[j]] + ([db[j]] if case["bias"] else [])
    return outs
