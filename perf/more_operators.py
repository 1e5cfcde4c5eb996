"""What a training step needs around the bf16 expert layer, and the way of its weights back into the 4-bit format that
is served, as cases that can be timed.

  fp4_linear       ops.fp4_linear: x in bf16 is quantised to e2m1 codes with one power of two per 32 values, as the
                   weights are already, and multiplied by them
  embed            ops.embed: scale * table[id]; an id outside the table gives a row of zeros
  embed_grad       ops.embed_grad: the table's gradient, every row of the table written
  block_norm       ops.block_norm: h' = h + scale * gate * norm(f) after a block f, and norm(h') before the next one
  block_norm_grad  ops.block_norm_grad: the gradient of f, h, the gate and both norms' weights
  clip             ops.clip_grads: the norm of all gradients, and the gradients cut down to a limit on it
Sizes are those of MoEConfig (hidden 4096, expert 2048, vocabulary 129280, 256 experts) and, among the drawn ones,
generic ones.
"""
import math

import torch

own = False  # True: the framework's operators, False: their plain form

DEVICE = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


def listed():
    return [
        # a projection of one decoded token: the weights' stream, and the launches
        {"name": "fp4_linear_1", "kind": "fp4_linear", "m": 1, "n": 4096, "kk": 4096},
        # sequences that decode together
        {"name": "fp4_linear_33", "kind": "fp4_linear", "m": 33, "n": 4096, "kk": 4096},
        # a ragged prompt through an expert's gate: few tiles
        {"name": "fp4_linear_500", "kind": "fp4_linear", "m": 500, "n": 2048, "kk": 4096},
        # a square projection of a long ragged batch: the matrix cores
        {"name": "fp4_linear_8190", "kind": "fp4_linear", "m": 8190, "n": 4096, "kk": 4096},
        # a token and its drafts looked up: latency
        {"name": "embed_5", "kind": "embed", "m": 5, "vocab": 129280, "d": 4096, "type": "bf16", "ids": "int64",
         "scale": 64.0, "zipf": 1.0, "outside": 0.0},
        # the batch of a training step, with padding ids
        {"name": "embed_16381", "kind": "embed", "m": 16381, "vocab": 129280, "d": 4096, "type": "bf16",
         "ids": "int64", "scale": 64.0, "zipf": 1.0, "outside": 0.05},
        # its backward pass: a few words make up much of the batch, most of the table is not met
        {"name": "embed_grad_16381", "kind": "embed_grad", "m": 16381, "vocab": 129280, "d": 4096, "type": "bf16",
         "ids": "int64", "scale": 64.0, "zipf": 1.0, "outside": 0.05},
        # a verify's three tokens between two layers: latency
        {"name": "block_norm_3", "kind": "block_norm", "m": 3, "d": 4096, "type": "bf16", "stream": "bf16",
         "gate": "channel", "post": True, "pre": True, "scale": 0.5},
        # a training step's tokens between two layers, everything on
        {"name": "block_norm_8191", "kind": "block_norm", "m": 8191, "d": 4096, "type": "bf16", "stream": "f32",
         "gate": "full", "post": True, "pre": True, "scale": 0.5},
        # and their way back
        {"name": "block_norm_grad_8191", "kind": "block_norm_grad", "m": 8191, "d": 4096, "type": "bf16",
         "stream": "bf16", "gate": "channel", "post": True, "pre": True, "scale": 0.5},
        # the small gradients of a layer that is tuned by its norms and router alone: latency
        {"name": "clip_norms", "kind": "clip", "tensors": 6, "largest": 4096, "ratio": 0.5, "types": "f32",
         "out": "f32", "norm": 2.0, "max_norm": 1.0},
        # the gradients of all experts here and what stands around them, many sizes
        {"name": "clip_experts", "kind": "clip", "tensors": 60, "largest": 134217728, "ratio": 0.75, "types": "mixed",
         "out": "same", "norm": 2.0, "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("fp4_linear", "fp4_linear", "fp4_linear", "embed", "embed_grad", "block_norm",
                       "block_norm_grad", "clip"))
    case = {"kind": kind}
    if kind == "fp4_linear":
        case.update(m=_log_int(rng, 1, 8192), n=8 * _log_int(rng, 8, 512), kk=32 * _log_int(rng, 2, 128))
    elif kind in ("embed", "embed_grad"):
        case.update(m=_log_int(rng, 1, 16384), vocab=_log_int(rng, 100, 129280),
                    d=rng.choice((8 * _log_int(rng, 8, 512), _log_int(rng, 64, 4096), 4096)),
                    type=rng.choice(("bf16", "bf16", "f32")), ids=rng.choice(("int64", "int64", "int32")),
                    scale=rng.choice((1.0, round(rng.uniform(0.01, 64.0), 3))), zipf=round(rng.uniform(0.0, 1.3), 2),
                    outside=rng.choice((0.0, 0.0, round(rng.uniform(0.0, 0.9), 2))))
        if case["type"] == "f32":  # no more than the largest listed table's bytes
            case["vocab"] = min(case["vocab"], 64640)
            case["m"] = min(case["m"], 8192)
    elif kind in ("block_norm", "block_norm_grad"):
        case.update(m=_log_int(rng, 1, 8192), d=8 * _log_int(rng, 8, 1024), type=rng.choice(("bf16", "bf16", "f32")),
                    stream=rng.choice(("bf16", "f32")), gate=rng.choice(("none", "channel", "token", "full")),
                    post=rng.random() < 0.7, pre=rng.random() < 0.7, scale=rng.choice((1.0, 0.5, round(rng.random(), 3))))
        while case["m"] * case["d"] > 8191 * 4096 // (2 if case["type"] == "f32" else 1):
            case["m"] = (case["m"] + 1) // 2
    else:
        types = rng.choice(("bf16", "f32", "mixed"))
        case.update(tensors=_log_int(rng, 1, 60), largest=_log_int(rng, 1, 1 << 26), ratio=round(rng.uniform(0.3, 1.0), 3),
                    types=types, out=rng.choice(("same", "f32")), norm=rng.choice((2.0, 2.0, math.inf)),
                    max_norm=rng.choice((1.0, round(rng.uniform(0.1, 10.0), 3), 1e9)))
        while work(case)["bytes"] > 2e9:
            case["largest"] = (case["largest"] + 1) // 2
    return case


# ---------------------------------------------------------------- inputs

def _gen(seed, sub):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 64 + sub)
    return g


def _normal(seed, sub, shape, std, dtype=BF16, mean=0.0):
    t = torch.randn(shape, generator=_gen(seed, sub), device=DEVICE, dtype=dtype).mul_(std)
    return t.add_(mean) if mean else t


def _dtype(name):
    return F32 if name == "f32" else BF16


def _ids(case, seed):
    """Popularity falls as 1 / rank^zipf; a share of the ids is -1 (padding) or behind the table."""
    v, m = case["vocab"], case["m"]
    p = torch.arange(1, v + 1, device=DEVICE, dtype=F64) ** -case["zipf"]
    cum = (p / p.sum()).cumsum(0)
    u = torch.rand(m, generator=_gen(seed, 1), device=DEVICE, dtype=F64)
    rank = torch.searchsorted(cum, u).clamp_(max=v - 1)
    ids = torch.randperm(v, generator=_gen(seed, 2), device=DEVICE)[rank]
    if case["outside"]:
        o = torch.rand(m, generator=_gen(seed, 3), device=DEVICE)
        ids = torch.where(o < case["outside"], torch.where(o < case["outside"] / 4, v, -1), ids)
    return ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)


def _clip_shapes(case):
    """Tensor j: (elements, type name, out type name); sizes fall by `ratio`, those of one element at least."""
    shapes, n = [], float(case["largest"])
    for j in range(case["tensors"]):
        t = case["types"] if case["types"] != "mixed" else ("f32" if j % 4 == 3 else "bf16")
        shapes.append((max(1, int(n)), t, t if case["out"] == "same" else case["out"]))
        n *= case["ratio"]
        if n < 1.0:
            n = float(min(case["largest"], 4099))
    return shapes


def prepare(case, seed):
    """Inputs from the seed; weights quantised as they are kept; buffers for the clipped gradients."""
    kind = case["kind"]
    state = {"kind": kind, "case": case}
    if kind == "fp4_linear":
        m, n, kk = case["m"], case["n"], case["kk"]
        x = _normal(seed, 4, (m, kk), 1.0)
        # some channels of activations are far larger than the others
        loud = torch.rand(kk, generator=_gen(seed, 5), device=DEVICE) < 0.01
        state["x"] = torch.where(loud, x * 16, x)
        codes, scale = _quantise(_normal(seed, 6, (n, kk), 1.0 / math.sqrt(kk)))
        state["w"] = (codes[:, 0::2] | codes[:, 1::2] << 4).view(torch.int8)
        state["w_scale"] = scale.view(torch.float8_e8m0fnu)
    elif kind == "embed":
        state["ids"] = _ids(case, seed)
        state["table"] = _normal(seed, 4, (case["vocab"], case["d"]), 0.02, _dtype(case["type"]))
    elif kind == "embed_grad":
        state["ids"] = _ids(case, seed)
        state["d_out"] = _normal(seed, 4, (case["m"], case["d"]), 0.01, _dtype(case["type"]))
    elif kind in ("block_norm", "block_norm_grad"):
        m, d, t, s = case["m"], case["d"], _dtype(case["type"]), _dtype(case["stream"])
        state["f"] = _normal(seed, 4, (m, d), 3.0, t)
        state["h"] = _normal(seed, 5, (m, d), 2.0, s)  # the gradient takes the stream after the block
        if case["post"]:
            state["post_w"] = _normal(seed, 6, (d,), 0.1, t, 1.0)
        if case["pre"]:
            state["pre_w"] = _normal(seed, 7, (d,), 0.1, t, 1.0)
        if case["gate"] != "none":
            shape = {"channel": (d,), "token": (m, 1), "full": (m, d)}[case["gate"]]
            state["gate"] = _normal(seed, 8, shape, 0.3, t, 0.5)
        if kind == "block_norm_grad":
            state["d_h"] = _normal(seed, 9, (m, d), 1.0, s)
            if case["pre"]:
                state["d_n"] = _normal(seed, 10, (m, d), 1.0, t)
    else:
        shapes = _clip_shapes(case)
        state["grads"] = [_normal(seed, 4 + j, (n,), 0.02 * (1 + j % 7), _dtype(t)) for j, (n, t, _) in enumerate(shapes)]
        state["out"] = [torch.empty(n, device=DEVICE, dtype=_dtype(o)) for n, _, o in shapes]
    return state


# ---------------------------------------------------------------- the pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import __graft_entry__
    __graft_entry__.package()
    from home_seek_amd import ops

    kind, case = state["kind"], state["case"]
    if kind == "fp4_linear":
        return ops.fp4_linear(state["x"], state["w"], state["w_scale"])
    if kind == "embed":
        return ops.embed(state["ids"], state["table"], case["scale"])
    if kind == "embed_grad":
        return ops.embed_grad(state["d_out"], state["ids"], case["vocab"], case["scale"])
    if kind == "block_norm":
        h, n = ops.block_norm(state["f"], state["h"], state.get("post_w"), state.get("gate"), case["scale"],
                              state.get("pre_w"), EPS)
        return [h] if n is None else [h, n]
    if kind == "block_norm_grad":
        g = ops.block_norm_grad(state["d_h"], state.get("d_n"), state["f"], state["h"], state.get("post_w"),
                                state.get("gate"), case["scale"], state.get("pre_w"), EPS)
        return [t for t in g if t is not None]
    norm = ops.clip_grads(state["grads"], case["max_norm"], case["norm"], out=state["out"])
    return [norm] + state["out"]


def _quantise(x):
    """Codes (uint8, one each) and scale exponents (uint8, one per 32) of finite x: the scale is the smallest power of
    two with which the largest of its values is at most 6, the codes are the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6,
    ties to the even code."""
    blocks = x.float().reshape(x.shape[0], -1, 32)
    mant, exp = torch.frexp(blocks.abs().amax(dim=2))  # mant * 2^exp, mant in [0.5, 1)
    byte = (exp + torch.where(mant > 0.75, 125, 124)).clamp(0, 254)  # mant * 2^exp <= 0.75 * 2^3 * 2^(exp - 3)
    byte = torch.where(mant > 0, byte, 0)
    a = torch.ldexp(blocks, (127 - byte)[:, :, None])
    code = torch.zeros_like(blocks, dtype=torch.uint8)
    mag = a.abs()
    for limit, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (mag >= limit) if tie_up else (mag > limit)
    code = torch.where(torch.signbit(a), code | 8, code)
    return code.reshape(x.shape), byte.to(torch.uint8)


_CODE_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(codes, byte, dtype):
    """What codes and exponents stand for."""
    table = torch.tensor(_CODE_VALUES + tuple(-v for v in _CODE_VALUES), dtype=dtype, device=codes.device)
    v = table[codes.long()].reshape(codes.shape[0], -1, 32)
    return torch.ldexp(v, byte.to(torch.int32)[:, :, None] - 127).reshape(codes.shape)


def _rms(t):
    return torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS)


def _run_plain(state):
    kind, case = state["kind"], state["case"]
    if kind == "fp4_linear":
        x = _values(*_quantise(state["x"]), F32)
        b = state["w"].view(torch.uint8)
        w = _values(torch.stack((b & 15, b >> 4), dim=2).reshape(case["n"], case["kk"]),
                    state["w_scale"].view(torch.uint8), F32)
        return (x @ w.T).to(BF16)
    if kind == "embed":
        ids, v = state["ids"].long(), case["vocab"]
        inside = (ids >= 0) & (ids < v)
        rows = state["table"][torch.where(inside, ids, 0)]
        return torch.where(inside[:, None], rows.float() * case["scale"], 0.0).to(rows.dtype)
    if kind == "embed_grad":
        ids, v, d_out = state["ids"].long(), case["vocab"], state["d_out"]
        inside = (ids >= 0) & (ids < v)
        dw = torch.zeros(v + 1, case["d"], dtype=F32, device=DEVICE)
        dw.index_add_(0, torch.where(inside, ids, v), d_out.float())
        return (dw[:v] * case["scale"]).to(d_out.dtype)
    if kind == "block_norm":
        f, h = state["f"].float(), state["h"]
        u = f * _rms(f) * state["post_w"].float() if case["post"] else f
        if case["gate"] != "none":
            u = u * state["gate"].float()
        h2 = (h.float() + case["scale"] * u).to(h.dtype)
        if not case["pre"]:
            return [h2]
        t = h2.float()
        return [h2, (t * _rms(t) * state["pre_w"].float()).to(state["f"].dtype)]
    if kind == "block_norm_grad":
        f, dh = state["f"].float(), state["d_h"].float()
        outs = {}
        if case["pre"]:
            h, dn = state["h"].float(), state["d_n"].float()
            r = _rms(h)
            y = h * r
            outs["pre_w"] = (dn * y).sum(dim=0)
            dy = dn * state["pre_w"].float()
            dh = dh + r * (dy - y * (dy * y).mean(dim=1, keepdim=True))
        outs["h"] = dh.to(state["h"].dtype)
        du = case["scale"] * dh
        r = _rms(f)
        y = f * r
        u = y * state["post_w"].float() if case["post"] else f
        if case["gate"] != "none":
            dg = du * u
            outs["gate"] = {"channel": lambda: dg.sum(dim=0), "token": lambda: dg.sum(dim=1, keepdim=True),
                            "full": lambda: dg.to(state["gate"].dtype)}[case["gate"]]()
            du = du * state["gate"].float()
        if case["post"]:
            outs["post_w"] = (du * y).sum(dim=0)
            du = du * state["post_w"].float()
            du = r * (du - y * (du * y).mean(dim=1, keepdim=True))
        outs["f"] = du.to(state["f"].dtype)
        return [outs[k] for k in ("f", "h", "post_w", "gate", "pre_w") if k in outs]
    if case["norm"] == 2.0:
        norm = sum((g.float() ** 2).sum() for g in state["grads"]).sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in state["grads"]]).max()
    c = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, o in zip(state["grads"], state["out"]):
        o.copy_(g.float() * c)
    return [norm] + state["out"]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "f32": 4}
    if kind == "fp4_linear":
        m, n, kk = case["m"], case["n"], case["kk"]
        return {"bytes": 2.0 * m * kk + n * kk * 17 / 32 + 2.0 * m * n, "flops": 2.0 * m * n * kk}
    if kind in ("embed", "embed_grad"):
        m, v, d, s = case["m"], case["vocab"], case["d"], size[case["type"]]
        live = m * (1.0 - case["outside"])
        ids = m * (4 if case["ids"] == "int32" else 8)
        if kind == "embed_grad":
            return {"bytes": ids + live * d * s + float(v) * d * s, "flops": live * d}
        p = torch.arange(1, v + 1, dtype=F64) ** -case["zipf"]
        met = float((1.0 - (1.0 - p / p.sum()) ** live).sum())  # rows that are looked up at least once, on average
        return {"bytes": ids + met * d * s + float(m) * d * s, "flops": live * d}
    if kind in ("block_norm", "block_norm_grad"):
        md, t, s = float(case["m"] * case["d"]), size[case["type"]], size[case["stream"]]
        gate = t * md if case["gate"] == "full" else 0.0
        if kind == "block_norm":
            return {"bytes": md * (t + 2 * s) + gate + (md * t if case["pre"] else 0.0), "flops": 10.0 * md}
        nbytes = md * (2 * t + 2 * s) + 2 * gate + (md * (s + t) if case["pre"] else 0.0)
        return {"bytes": nbytes, "flops": 24.0 * md}
    nbytes = sum(n * (size[t] + size[o]) for n, t, o in _clip_shapes(case))
    return {"bytes": float(nbytes), "flops": 3.0 * sum(n for n, _, _ in _clip_shapes(case))}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """From the definitions, in 64 bits."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "fp4_linear":
        m, n, kk = case["m"], case["n"], case["kk"]
        grid = torch.tensor(_CODE_VALUES, dtype=F64, device=DEVICE)
        x = state["x"].double().reshape(m * kk // 32, 32)
        # the power of two, found by trying: doubled until the largest fits
        top = x.abs().max(dim=1, keepdim=True).values
        e = torch.full_like(top, -127.0)
        e = torch.where(top > 0, torch.maximum(e, torch.ceil(torch.log2(top.clamp(min=1e-300) / 6.0)) - 1), e)
        for _ in range(2):
            e = torch.where(6.0 * torch.exp2(e) < top, e + 1, e)
        v = x / torch.exp2(e)
        near = torch.empty_like(v)
        for a in range(0, v.shape[0], 1 << 18):
            part = v[a:a + (1 << 18)].abs()
            dist = (part[:, :, None] - grid).abs()
            best = dist.min(dim=2, keepdim=True).values
            even = (dist == best) & (torch.arange(8, device=DEVICE) % 2 == 0)
            pick = torch.where(even.any(dim=2), even.int().argmax(dim=2), (dist == best).int().argmax(dim=2))
            near[a:a + (1 << 18)] = grid[pick]
        x = (torch.sign(v) * near * torch.exp2(e)).reshape(m, kk)
        b = state["w"].to(torch.int32) & 255
        w = torch.zeros(n, kk, dtype=F64, device=DEVICE)
        for j, nib in enumerate((b % 16, b // 16)):
            w[:, j::2] = grid[nib % 8] * torch.where(nib >= 8, -1.0, 1.0).double()
        w = w * torch.exp2(state["w_scale"].view(torch.uint8).double() - 127).repeat_interleave(32, dim=1)
        return torch.matmul(x, w.t())
    if kind == "embed":
        out = torch.zeros(case["m"], case["d"], dtype=F64, device=DEVICE)
        t = torch.nonzero((state["ids"] >= 0) & (state["ids"] < case["vocab"]))[:, 0]
        out[t] = state["table"][state["ids"][t].long()].double() * case["scale"]
        return out
    if kind == "embed_grad":
        t = torch.nonzero((state["ids"] >= 0) & (state["ids"] < case["vocab"]))[:, 0]
        ids = state["ids"][t].long()
        dw = torch.zeros(case["vocab"], case["d"], dtype=F64, device=DEVICE)
        dw.index_put_((ids,), state["d_out"][t].double() * case["scale"], accumulate=True)
        return dw
    if kind in ("block_norm", "block_norm_grad"):
        f, h, d = state["f"].double(), state["h"].double(), case["d"]
        gate = state["gate"].double() if "gate" in state else torch.ones(1, dtype=F64, device=DEVICE)
        r1 = (f.pow(2).sum(dim=1, keepdim=True) / d + EPS).pow(-0.5)
        w1 = state["post_w"].double() if case["post"] else None
        u = f if w1 is None else f * r1 * w1
        if kind == "block_norm":
            h2 = h + case["scale"] * gate * u
            if not case["pre"]:
                return [h2]
            h3 = h2.to(state["h"].dtype).double()  # the stream is held in its type, and the norm is of what is held
            r2 = (h3.pow(2).sum(dim=1, keepdim=True) / d + EPS).pow(-0.5)
            return [h2, h3 * r2 * state["pre_w"].double()]
        dh = state["d_h"].double()
        d_pre = None
        if case["pre"]:
            r2 = (h.pow(2).sum(dim=1, keepdim=True) / d + EPS).pow(-0.5)
            dn = state["d_n"].double()
            d_pre = (dn * h * r2).sum(dim=0)
            g = dn * state["pre_w"].double()
            dh = dh + g * r2 - h * r2.pow(3) * (g * h).sum(dim=1, keepdim=True) / d
        dt = dh * case["scale"]
        du = dt * gate
        df, d_post = du, None
        if w1 is not None:
            d_post = (du * f * r1).sum(dim=0)
            g = du * w1
            df = g * r1 - f * r1.pow(3) * (g * f).sum(dim=1, keepdim=True) / d
        outs = [df, dh] + ([d_post] if d_post is not None else [])
        if case["gate"] != "none":
            dg = dt * u
            outs.append({"channel": dg.sum(dim=0), "token": dg.sum(dim=1, keepdim=True), "full": dg}[case["gate"]])
        return outs + ([d_pre] if d_pre is not None else [])
    if case["norm"] == 2.0:
        total = torch.zeros((), dtype=F64, device=DEVICE)
        for g in state["grads"]:
            total = total + torch.dot(g.double(), g.double())
        norm = torch.sqrt(total)
    else:
        norm = max(g.double().abs().max() for g in state["grads"])
    c = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    return [norm] + [g.double() * c for g in state["grads"]]
