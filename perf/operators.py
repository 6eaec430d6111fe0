"""The mixture-of-experts operators and the 8-bit products as they are measured.

    route           logits -> the top-k experts of each token and their weights (and d logits)
    experts         the routed SwiGLU experts in 16 bits, forward and training step
    fp8_linear      product in 8-bit floating point with a scale for each block of 128
    fp8_experts     the routed SwiGLU experts on 8-bit weights, for serving

``run`` computes an operator in plain torch operations, or, with ``own`` set, through the
package's public calls; ``exact`` computes it once more in 64 bits from the definition.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------- cases --
def listed():
    return [
        # one token of a small batch-1 decoder: all launch latency
        dict(name="route_token", op="route", T=1, E=64, k=6, dtype="bf16", score="softmax", bias=False,
             groups=1, topk_groups=1, renorm=True, scale=1.0, train=False),
        # a long prompt through a router with balance bias and expert groups
        dict(name="route_prompt", op="route", T=16384, E=256, k=8, dtype="fp32", score="sigmoid", bias=True,
             groups=8, topk_groups=4, renorm=True, scale=2.5, train=False),
        # a training step's routing, ragged number of tokens, plain softmax weights
        dict(name="route_train", op="route", T=8191, E=128, k=8, dtype="bf16", score="softmax", bias=False,
             groups=1, topk_groups=1, renorm=False, scale=1.0, train=True),
        # decoding one token: reads the weights of its k experts
        dict(name="experts_token", op="experts", T=1, E=64, k=6, d=4096, f=1408, dtype="bf16", train=False),
        # a prompt over many small experts
        dict(name="experts_prompt", op="experts", T=2047, E=64, k=6, d=4096, f=1408, dtype="bf16", train=False),
        # training step, few large experts (the 8B MLP shape as experts)
        dict(name="experts_train", op="experts", T=8192, E=8, k=2, d=4096, f=14336, dtype="bf16", train=True),
        # training step, odd sizes, more experts than some batches fill
        dict(name="experts_train_odd", op="experts", T=1001, E=60, k=4, d=1032, f=712, dtype="fp16", train=True),
        # decoding one token through a gate/up projection of the 8B shape
        dict(name="fp8_token", op="fp8_linear", T=1, d=4096, n=14336, dtype="bf16"),
        # a small odd batch through a down projection: few output tiles, long inner size
        dict(name="fp8_batch", op="fp8_linear", T=77, d=14336, n=4104, dtype="fp16"),
        # a prompt
        dict(name="fp8_prompt", op="fp8_linear", T=8192, d=4096, n=14336, dtype="bf16"),
        # decoding four tokens over 8-bit experts
        dict(name="fp8_experts_token", op="fp8_experts", T=4, E=64, k=6, d=4096, f=1408, dtype="bf16"),
        # a prompt over 8-bit experts
        dict(name="fp8_experts_prompt", op="fp8_experts", T=4096, E=64, k=6, d=4096, f=1408, dtype="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["route", "route", "experts", "experts", "fp8_linear", "fp8_experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log(rng, 4, 64)
        topk_groups = rng.randint(1, groups)
        k = rng.randint(1, min(12, topk_groups * (E // groups)))
        return dict(op=op, T=_log(rng, 1, 16384), E=E, k=k, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    topk_groups=topk_groups, renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]),
                    train=rng.random() < 0.5)
    if op == "fp8_linear":
        return dict(op=op, T=_log(rng, 1, 8192), d=_log(rng, 128, 14336, 16), n=_log(rng, 128, 14336, 8),
                    dtype=rng.choice(["bf16", "fp16"]))
    E = _log(rng, 4, 64)
    k = rng.randint(1, min(8, E))
    T = _log(rng, 1, 4096)
    train = op == "experts" and rng.random() < 0.5
    case = dict(op=op, T=T, E=E, k=k, d=_log(rng, 256, 4096, 16), f=_log(rng, 256, 2048, 16),
                dtype=rng.choice(["bf16", "fp16"]))
    if op == "experts":
        case["train"] = train
    return case


def work(case):
    T = case["T"]
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        size = 4 if case["dtype"] == "fp32" else 2
        nbytes = T * E * size + T * k * 8 + (E * 4 if case["bias"] else 0)
        flops = T * E * 8
        if case["train"]:
            nbytes += T * k * 4 + T * E * size
            flops += T * E * 4
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "fp8_linear":
        d, n = case["d"], case["n"]
        blocks = -(-d // 128) * -(-n // 128)
        return {"bytes": T * d * 2 + n * d + blocks * 4 + T * n * 2, "flops": 2 * T * n * d}
    E, k, d, f = case["E"], case["k"], case["d"], case["f"]
    used = min(E, T * k)
    flops = 6 * T * k * d * f
    if case["op"] == "fp8_experts":
        return {"bytes": used * 3 * d * f + 2 * T * d * 2 + T * k * 8, "flops": flops}
    nbytes = used * 3 * d * f * 2 + 2 * T * d * 2 + T * k * 8
    if case["train"]:
        nbytes += E * 3 * d * f * 2 + 2 * T * d * 2 + T * k * 2
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# -------------------------------------------------------------------------------- state --
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _routing(case, g):
    """Indices and weights of a router whose experts are unevenly popular."""
    T, E, k = case["T"], case["E"], case["k"]
    popular = torch.randn(E, device=DEV, generator=g) * 0.5
    logits = torch.randn(T, E, device=DEV, generator=g) + popular
    top, idx = torch.topk(logits, k, dim=1)
    return torch.softmax(top, dim=1).to(TYPES[case["dtype"]]), idx.to(torch.int32)


def _fp8_weight(rows, cols, g, experts=None):
    """An 8-bit checkpoint's weight (out, in) with one fp32 scale for each 128 x 128 block."""
    if experts is not None:
        pairs = [_fp8_weight(rows, cols, g) for _ in range(experts)]
        return torch.stack([q for q, _ in pairs]), torch.stack([s for _, s in pairs])
    w = torch.randn(rows, cols, device=DEV, generator=g) / math.sqrt(cols)
    rb, cb = -(-rows // 128), -(-cols // 128)
    pad = torch.zeros(rb * 128, cb * 128, device=DEV)
    pad[:rows, :cols] = w
    blocks = pad.view(rb, 128, cb, 128)
    scale = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (blocks / scale[:, None, :, None]).view(rb * 128, cb * 128)[:rows, :cols]
    return q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).contiguous(), scale


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    T = case["T"]
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        dt = TYPES[case["dtype"]]
        popular = torch.randn(E, device=DEV, generator=g) * 0.5
        st["logits"] = (torch.randn(T, E, device=DEV, generator=g) + popular).to(dt)
        # a balance bias moves in equal small steps, so many experts share a value
        st["bias"] = (torch.randn(E, device=DEV, generator=g) * 8).round() * 1e-3 if case["bias"] else None
        if case["train"]:
            st["dweights"] = torch.randn(T, k, device=DEV, generator=g)
            st["logits"].requires_grad_(True)
        return st
    dt = TYPES[case["dtype"]]
    d = case["d"]
    st["x"] = torch.randn(T, d, device=DEV, generator=g).to(dt)
    if case["op"] == "fp8_linear":
        st["w"], st["ws"] = _fp8_weight(case["n"], d, g)
        return st
    E, f = case["E"], case["f"]
    st["weights"], st["indices"] = _routing(case, g)
    if case["op"] == "fp8_experts":
        st["wg"], st["wgs"] = _fp8_weight(f, d, g, E)
        st["wu"], st["wus"] = _fp8_weight(f, d, g, E)
        st["wd"], st["wds"] = _fp8_weight(d, f, g, E)
        return st
    for name, rows, cols in (("wg", d, f), ("wu", d, f), ("wd", f, d)):
        w = torch.empty(E, rows, cols, device=DEV, dtype=dt)
        for e in range(E):
            w[e] = torch.randn(rows, cols, device=DEV, generator=g) / math.sqrt(rows)
        st[name] = w
    if case["train"]:
        st["dy"] = torch.randn(T, d, device=DEV, generator=g).to(dt)
        for name in ("x", "weights", "wg", "wu", "wd"):
            st[name].requires_grad_(True)
    return st


# ------------------------------------------------------------------- the package's calls --
def _run_own(st):
    import fusedswiglu_b200 as fsw

    case = st["case"]
    if case["op"] == "route":
        w, idx = fsw.route(st["logits"], case["k"], bias=st["bias"], score=case["score"],
                           renormalize=case["renorm"], scale=case["scale"], num_groups=case["groups"],
                           topk_groups=case["topk_groups"])
        if not case["train"]:
            return [w, idx]
        (dl,) = torch.autograd.grad(w, [st["logits"]], st["dweights"])
        return [w.detach(), idx, dl]
    if case["op"] == "fp8_linear":
        return [fsw.fp8_linear(st["x"], st["w"], st["ws"])]
    if case["op"] == "fp8_experts":
        return [fsw.fp8_swiglu_experts(st["x"], st["weights"], st["indices"], st["wg"], st["wgs"], st["wu"],
                                       st["wus"], st["wd"], st["wds"])]
    y = fsw.FusedSwiGLUExperts.apply(st["x"], st["weights"], st["indices"], st["wg"], st["wu"], st["wd"])
    if not case["train"]:
        return [y]
    leaves = [st[n] for n in ("x", "weights", "wg", "wu", "wd")]
    return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]


# --------------------------------------------------------------------------- plain forms --
def _first_k(keys, k):
    """Indices of the k largest along the last axis, ties to the lowest index."""
    return torch.sort(keys, dim=-1, descending=True, stable=True).indices[..., :k]


def _route_plain(st):
    case = st["case"]
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    z = st["logits"].detach().double()  # selection: values next to a border
    s = torch.softmax(z, dim=1) if case["score"] == "softmax" else torch.sigmoid(z)
    choice = s + st["bias"].double() if st["bias"] is not None else s
    # without a bias the scores order as the logits do
    order = choice if st["bias"] is not None else z
    if G > 1:
        per = choice.view(T, G, E // G)
        best = torch.topk(per, min(2, E // G), dim=2).values.sum(dim=2)
        chosen = _first_k(best, case["topk_groups"])
        keep = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, chosen, True)
        order = order.masked_fill(~keep.repeat_interleave(E // G, dim=1), -math.inf)
    idx = _first_k(order, k)
    sel = torch.gather(s, 1, idx).float()
    total = sel.sum(dim=1, keepdim=True)
    w = (sel / total if case["renorm"] else sel) * case["scale"]
    if not case["train"]:
        return [w, idx.to(torch.int32)]
    dw = st["dweights"] * case["scale"]
    if case["renorm"]:
        part = sel / total
        ds = (dw - (part * dw).sum(dim=1, keepdim=True)) / total
    else:
        ds = dw
    s32 = s.float()
    full = torch.zeros(T, E, device=DEV).scatter_(1, idx, ds)
    if case["score"] == "softmax":
        dl = s32 * (full - (sel * ds).sum(dim=1, keepdim=True))
        if case["renorm"]:
            dl = dl * torch.zeros(T, E, device=DEV).scatter_(1, idx, 1.0)
    else:
        dl = full * s32 * (1.0 - s32)
    return [w, idx.to(torch.int32), dl.to(st["logits"].dtype)]


def _experts_plain(st):
    case = st["case"]
    dt = TYPES[case["dtype"]]
    x = st["x"].detach().float()
    weights = st["weights"].detach().float()
    y = torch.zeros_like(x)
    train = case["train"]
    if train:
        dy = st["dy"].float()
        dx, dweights = torch.zeros_like(x), torch.zeros_like(weights)
        dwg, dwu, dwd = (torch.zeros_like(st[n]) for n in ("wg", "wu", "wd"))
    for e in range(case["E"]):
        tok, slot = torch.nonzero(st["indices"] == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        wg, wu, wd = (st[n][e].detach().float() for n in ("wg", "wu", "wd"))
        xe, we = x[tok], weights[tok, slot][:, None]
        g, u = xe @ wg, xe @ wu
        sg = 1.0 / (1.0 + torch.exp(-g))
        h = g * sg * u
        y.index_add_(0, tok, we * (h @ wd))
        if train:
            dh = dy[tok] @ wd.t()
            dweights[tok, slot] = (dh * h).sum(dim=1)
            dh = dh * we
            du = dh * g * sg
            dg = dh * u * (sg + g * sg * (1.0 - sg))
            dx.index_add_(0, tok, dg @ wg.t() + du @ wu.t())
            dwg[e] = (xe.t() @ dg).to(dt)
            dwu[e] = (xe.t() @ du).to(dt)
            dwd[e] = (h.t() @ (we * dy[tok])).to(dt)
    if not train:
        return [y.to(dt)]
    return [y.to(dt), dx.to(dt), dweights.to(dt), dwg, dwu, dwd]


def _fp8_rows(x):
    """Values that rows hold after rounding to e4m3 with a power-of-two scale for each 128:
    the smallest one under which the largest magnitude fits."""
    T, d = x.shape
    nb = -(-d // 128)
    pad = torch.zeros(T, nb * 128, device=x.device, dtype=torch.float32)
    pad[:, :d] = x
    blocks = pad.view(T, nb, 128)
    m, ex = torch.frexp(blocks.abs().amax(dim=2))
    ex = torch.where(m > 0.875, ex - 8, ex - 9)
    scale = torch.where(m > 0, torch.ldexp(torch.ones_like(m), ex), torch.ones_like(m))
    q = (blocks / scale[:, :, None]).to(torch.float8_e4m3fn).float()
    return (q * scale[:, :, None]).view(T, nb * 128)[:, :d]


def _fp8_values(w, ws):
    rows, cols = w.shape
    full = ws.repeat_interleave(128, dim=0)[:rows].repeat_interleave(128, dim=1)[:, :cols]
    return w.float() * full


def _fp8_experts_plain(st):
    case = st["case"]
    x = _fp8_rows(st["x"].float())
    weights = st["weights"].float()
    y = torch.zeros_like(x)
    for e in range(case["E"]):
        tok, slot = torch.nonzero(st["indices"] == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        g = x[tok] @ _fp8_values(st["wg"][e], st["wgs"][e]).t()
        u = x[tok] @ _fp8_values(st["wu"][e], st["wus"][e]).t()
        h = _fp8_rows(g / (1.0 + torch.exp(-g)) * u)
        y.index_add_(0, tok, weights[tok, slot][:, None] * (h @ _fp8_values(st["wd"][e], st["wds"][e]).t()))
    return [y.to(TYPES[case["dtype"]])]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "route":
        return _route_plain(state)
    if op == "experts":
        return _experts_plain(state)
    if op == "fp8_linear":
        y = _fp8_rows(state["x"].float()) @ _fp8_values(state["w"], state["ws"]).t()
        return [y.to(TYPES[state["case"]["dtype"]])]
    return _fp8_experts_plain(state)


# ----------------------------------------------------------------- definition in 64 bits --
def _silu64(v):
    return v * torch.special.expit(v)


def _quantised64(v):
    """e4m3 values of rows in 64 bits, from the type's definition: 4 bits of significand
    down to 2**-6, steps of 2**-9 below, scaled by a power of two for each 128."""
    T, d = v.shape
    out = torch.empty_like(v)
    for c in range(0, d, 128):
        b = v[:, c:c + 128]
        top = b.abs().amax(dim=1, keepdim=True)
        power = torch.ceil(torch.log2(top / E4M3_MAX))
        power = torch.where(top > E4M3_MAX * 2.0 ** power, power + 1, power)
        power = torch.where(top <= E4M3_MAX * 2.0 ** (power - 1), power - 1, power)
        unit = torch.where(top > 0, 2.0 ** power, torch.ones_like(top))
        r = b / unit
        step = 2.0 ** (torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, c:c + 128] = torch.round(r / step) * step * unit
    return out


def _weight64(w, ws):
    out = w.to(torch.float64)
    for i in range(ws.shape[0]):
        for j in range(ws.shape[1]):
            out[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= ws[i, j].double()
    return out


def _exact_route(st):
    case = st["case"]
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    z = st["logits"].detach().double()
    if case["score"] == "softmax":
        p = torch.exp(z - z.amax(dim=1, keepdim=True))
        s = p / p.sum(dim=1, keepdim=True)
    else:
        s = torch.special.expit(z)
    c = s if st["bias"] is None else s + st["bias"].double()
    rank_by = z.clone() if st["bias"] is None else c.clone()
    rows = torch.arange(T, device=DEV)
    if G > 1:
        size = E // G
        two = torch.sort(c.view(T, G, size), dim=2, descending=True).values[:, :, :2].sum(dim=2)
        allowed = torch.zeros(T, G, dtype=torch.bool, device=DEV)
        for _ in range(case["topk_groups"]):
            best = torch.where(allowed, -math.inf, two)
            # the first group that reaches the maximum
            at = (best == best.amax(dim=1, keepdim=True)).int().argmax(dim=1)
            allowed[rows, at] = True
        for grp in range(G):
            block = rank_by[:, grp * size:(grp + 1) * size]
            block[~allowed[:, grp]] = -math.inf
    picks = []
    for _ in range(k):
        at = (rank_by == rank_by.amax(dim=1, keepdim=True)).int().argmax(dim=1)
        picks.append(at)
        rank_by[rows, at] = -math.inf
    idx = torch.stack(picks, dim=1)
    z2 = z.clone().requires_grad_(True)
    s2 = torch.softmax(z2, dim=1) if case["score"] == "softmax" else torch.special.expit(z2)
    w = torch.gather(s2, 1, idx)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    w = w * case["scale"]
    if not case["train"]:
        return [w.detach(), idx.to(torch.int32)]
    (dl,) = torch.autograd.grad(w, [z2], st["dweights"].double())
    return [w.detach(), idx.to(torch.int32), dl]


def _exact_experts(st):
    case = st["case"]
    eight = case["op"] == "fp8_experts"
    train = case.get("train", False)
    x = st["x"].detach().double()
    if eight:
        x = _quantised64(x)
    r = st["weights"].detach().double()
    y = torch.zeros_like(x)
    if train:
        dy = st["dy"].double()
        dx, dr = torch.zeros_like(x), torch.zeros_like(r)
        grads = {n: torch.zeros(st[n].shape, dtype=torch.float32, device=DEV) for n in ("wg", "wu", "wd")}
    owner = st["indices"].long()
    for e in range(case["E"]):
        hit = (owner == e).nonzero()
        if hit.shape[0] == 0:
            continue
        t, j = hit[:, 0], hit[:, 1]
        if eight:
            a, b, c = (_weight64(st[n][e], st[n + "s"][e]).t() for n in ("wg", "wu", "wd"))
        else:
            a, b, c = (st[n][e].detach().double() for n in ("wg", "wu", "wd"))
        if train:
            leaves = [v.clone().requires_grad_(True) for v in (x[t], r[t, j], a, b, c)]
            xi, ri, a, b, c = leaves
            out = ri[:, None] * ((_silu64(xi @ a) * (xi @ b)) @ c)
            gx, gr, ga, gb, gc = torch.autograd.grad(out, leaves, dy[t])
            dx.index_add_(0, t, gx)
            dr[t, j] = gr
            # kept in 32 bits for room; far finer than the 16-bit gradients they are held against
            grads["wg"][e], grads["wu"][e], grads["wd"][e] = ga.float(), gb.float(), gc.float()
            y.index_add_(0, t, out.detach())
        else:
            h = _silu64(x[t] @ a) * (x[t] @ b)
            if eight:
                h = _quantised64(h)
            y.index_add_(0, t, r[t, j][:, None] * (h @ c))
    return [y, dx, dr, grads["wg"], grads["wu"], grads["wd"]] if train else [y]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(st)
    if case["op"] == "fp8_linear":
        return [_quantised64(st["x"].double()) @ _weight64(st["w"], st["ws"]).t()]
    return _exact_experts(st)
