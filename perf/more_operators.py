"""The measured workloads of layers in 8-bit integers, dense and of experts.

  norm     the residual's addition and the RMS norm of a layer's input, out as int8 rows with a scale each
  product  int8 weights with a scale per row times int8 activations with a scale per token
  route    the experts of each token and their weights, from the router's logits
  up       the gate and up products of the tokens' experts, silu(gate) * up
  down     the down products of the tokens' experts, weighted and summed per token

Sizes of products are those of this repository's configurations and tests, or generic. A case fixes how much
there is to do; the seed only values and which experts.
"""
import math

import torch

own = False

F32, F16 = 0, 1
DTYPES = {"F32": torch.float32, "F16": torch.float16}
DEV = "cuda"
EPS = 1e-6


def _norm(name, dtype, rows, width, residual=True):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "width": width, "residual": residual}


def _product(name, rows, n, k, out="F32", add="none"):
    return {"name": name, "op": "product", "rows": rows, "n": n, "k": k, "out": out, "add": add}


def _route(name, dtype, rows, experts, top, scoring, bias=False, groups=1, top_groups=1, group_best=1):
    return {"name": name, "op": "route", "dtype": dtype, "rows": rows, "experts": experts, "top": top, "scoring": scoring,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_best": group_best}


def _up(name, rows, experts, top, n, k, pad=0):
    return {"name": name, "op": "up", "rows": rows, "experts": experts, "top": top, "n": n, "k": k, "pad": pad}


def _down(name, rows, experts, top, n, k, residual=True, pad=0):
    return {"name": name, "op": "down", "rows": rows, "experts": experts, "top": top, "n": n, "k": k,
            "residual": residual, "pad": pad}


def listed():
    return [
        # one token's hidden state before a layer: launch latency
        _norm("norm_one", "F32", 1, 2560),
        # a prompt's hidden states, the layer before wrote F16
        _norm("norm_prompt", "F16", 2048, 4096),
        # one token's FFN projection
        _product("product_one", 1, 9728, 2560),
        # a served batch of odd size, with the residual
        _product("product_batch", 61, 2560, 9728, add="residual"),
        # a prompt's FFN projection
        _product("product_prompt", 2048, 8192, 2048),
        # a long ragged prompt chunk through a wide projection, F16 out
        _product("product_long", 4099, 14336, 4096, out="F16"),
        # a few users' tokens: softmax scores, best 8 of 128
        _route("route_few", "F32", 5, 128, 8, "softmax"),
        # a prompt: sigmoid scores, a bias for balance, the best 4 of 8 groups
        _route("route_prompt", "F32", 8192, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, group_best=2),
        # a few users' tokens: nearly every slot an expert of its own
        _up("up_few", 5, 128, 8, 768, 2048),
        # a ragged prompt chunk over 128 experts, with padded tokens behind it
        _up("up_prompt", 1531, 128, 8, 768, 2048, pad=40),
        # a served batch: all experts are read, a few rows each
        _down("down_batch", 48, 128, 8, 2048, 768),
        # a ragged prompt chunk over 128 experts
        _down("down_prompt", 1531, 128, 8, 2048, 768, pad=40),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "product", "product", "route", "up", "up", "down", "down"])
    if op == "norm":
        case = _norm("", rng.choice(["F32", "F16"]), _log_uniform(rng, 1, 3000), 16 * _log_uniform(rng, 4, 512),
                     residual=rng.random() < 0.8)
    elif op == "product":
        while True:
            case = _product("", _log_uniform(rng, 1, 6000), _log_uniform(rng, 16, 15000), 16 * _log_uniform(rng, 4, 640),
                            out=rng.choice(["F32", "F32", "F16"]), add=rng.choice(["none", "none", "residual", "bias"]))
            if work(case)["flops"] <= 4.8e11:
                break
    elif op == "route":
        experts = rng.choice([4, 8, 16, 60, 64, 128, 160, 256, 384])
        groups = rng.choice([1, 1, 2, 4])
        top = rng.randint(1, min(experts // groups, 10))
        case = _route("", rng.choice(["F32", "F16"]), _log_uniform(rng, 1, 8192), experts, top,
                      rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                      top_groups=rng.randint(1, groups), group_best=rng.choice([1, 2]))
    else:
        while True:
            experts = rng.choice([4, 8, 16, 60, 64, 128])
            top = rng.randint(1, min(experts, 8))
            hidden, width = 16 * _log_uniform(rng, 8, 256), 16 * _log_uniform(rng, 8, 160)
            rows = _log_uniform(rng, 1, 1500)
            pad = rng.choice([0, 0, rng.randint(0, rows)])
            case = (_up("", rows, experts, top, width, hidden, pad) if op == "up" else
                    _down("", rows, experts, top, hidden, width, residual=rng.random() < 0.7, pad=pad))
            if work(case)["flops"] <= 7e10 and 2 * experts * hidden * width <= 5e8:
                break
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def _hidden(rows, width, gen):
    """Hidden states: normal values with a few channels far above the others."""
    x = torch.randn((rows, width), generator=gen, device=DEV)
    hot = torch.randint(0, width, (max(width // 200, 1),), generator=gen, device=DEV)
    x[:, hot] *= 12.0
    return x


def _int8_rows(shape, gen, spread):
    """int8 rows as quantizing normal values to their largest leaves them, and the rows' scales."""
    q = torch.randn(shape, generator=gen, device=DEV).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
    return q, spread / 127.0 * (0.5 + torch.rand(shape[:-1], generator=gen, device=DEV))


def _ids(case, gen):
    """The tokens' experts: some experts are chosen more often than others; padded tokens have none (-1)."""
    t, e, top = case["rows"], case["experts"], case["top"]
    liked = 0.4 * torch.randn((1, e), generator=gen, device=DEV)
    ids = torch.topk(liked + torch.randn((t, e), generator=gen, device=DEV), top, dim=1).indices.int()
    return torch.cat([ids, torch.full((case["pad"], top), -1, dtype=torch.int32, device=DEV)])


def _prepare_norm(case, gen):
    m, k = case["rows"], case["width"]
    return {"x": _hidden(m, k, gen).to(DTYPES[case["dtype"]]), "r": 3.0 * _hidden(m, k, gen) if case["residual"] else None,
            "w": 1.0 + 0.2 * torch.randn(k, generator=gen, device=DEV), "h": torch.empty((m, k), device=DEV),
            "q": torch.empty((m, k), dtype=torch.int8, device=DEV), "s": torch.empty(m, device=DEV)}


def _prepare_product(case, gen):
    m, n, k = case["rows"], case["n"], case["k"]
    w, ws = _int8_rows((n, k), gen, 0.08)
    x, xs = _int8_rows((m, k), gen, 4.0)
    add = {"none": None, "residual": (m, n), "bias": (n,)}[case["add"]]
    st = {"w": w, "ws": ws, "x": x, "xs": xs, "r": None if add is None else torch.randn(add, generator=gen, device=DEV),
          "y": torch.empty((m, n), dtype=DTYPES[case["out"]], device=DEV)}
    if own:
        import densecore_amd as dc
        st["ws_mem"] = torch.empty(max(dc.mul_mat_i8_workspace_size(m, n, k), 256), dtype=torch.uint8, device=DEV)
    return st


def _prepare_route(case, gen):
    m, e = case["rows"], case["experts"]
    x = 1.5 * torch.randn((m, e), generator=gen, device=DEV)
    return {"x": x.to(DTYPES[case["dtype"]]),
            "bias": 0.1 * torch.randn(e, generator=gen, device=DEV) if case["bias"] else None,
            "ids": torch.empty((m, case["top"]), dtype=torch.int32, device=DEV),
            "weights": torch.empty((m, case["top"]), device=DEV)}


def _prepare_up(case, gen):
    e, n, k = case["experts"], case["n"], case["k"]
    wg, wgs = _int8_rows((e, n, k), gen, 0.08)
    wu, wus = _int8_rows((e, n, k), gen, 0.08)
    ids = _ids(case, gen)
    x, xs = _int8_rows((len(ids), k), gen, 4.0)
    st = {"wg": wg, "wgs": wgs, "wu": wu, "wus": wus, "x": x, "xs": xs, "ids": ids,
          "h": torch.empty((ids.numel(), n), device=DEV)}
    if own:
        import densecore_amd as dc
        st["plan"] = torch.empty(dc.moe_plan_size(*ids.shape, e), dtype=torch.uint8, device=DEV)
    return st


def _prepare_down(case, gen):
    e, n, k = case["experts"], case["n"], case["k"]
    w, ws = _int8_rows((e, n, k), gen, 0.08)
    ids = _ids(case, gen)
    h, hs = _int8_rows((ids.numel(), k), gen, 2.0)
    weights = torch.softmax(torch.randn(ids.shape, generator=gen, device=DEV), 1)
    st = {"w": w, "ws": ws, "h": h, "hs": hs, "ids": ids, "weights": weights,
          "r": 3.0 * _hidden(len(ids), n, gen) if case["residual"] else None, "y": torch.empty((len(ids), n), device=DEV)}
    if own:
        import densecore_amd as dc
        st["plan"] = torch.empty(dc.moe_plan_size(*ids.shape, e), dtype=torch.uint8, device=DEV)
        st["ws_mem"] = torch.empty(max(dc.moe_down_i8_workspace_size(*ids.shape, n), 256), dtype=torch.uint8, device=DEV)
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    make = {"norm": _prepare_norm, "product": _prepare_product, "route": _prepare_route, "up": _prepare_up,
            "down": _prepare_down}[case["op"]]
    return {"case": case, **make(case, gen)}


# ---------------------------------------------------------------- one pass
def _run_norm(st):
    if own:
        import densecore_amd as dc
        h, q, s = dc.rms_norm_i8(st["x"], st["w"], EPS, r=st["r"], h=st["h"] if st["r"] is not None else None, q=st["q"],
                                 s=st["s"])
    else:
        h = st["x"].float() if st["r"] is None else st["x"].float() + st["r"]
        p = h.double() * st["w"].double()  # 64 bits: which step a value next to a border rounds to
        top = p.abs().amax(1, keepdim=True)
        q = torch.round(p * (127.0 / top)).to(torch.int8)
        s = (top / (127.0 * torch.sqrt(h.double().square().mean(1, keepdim=True) + EPS))).float().view(-1)
    values = q * s[:, None]  # what the rows stand for
    return [values, s] if st["r"] is None else [values, s, h]


def _run_product(st):
    case = st["case"]
    if own:
        import densecore_amd as dc
        return dc.mul_mat_i8(st["w"], st["ws"], st["x"], st["xs"], r=st["r"], y=st["y"], workspace=st["ws_mem"])
    y = torch.matmul(st["x"].float(), st["w"].float().t()) * st["ws"] * st["xs"][:, None]
    if st["r"] is not None:
        y = y + st["r"]
    return y.to(DTYPES[case["out"]])


def _run_route(st):
    case = st["case"]
    groups, top = case["groups"], case["top"]
    if own:
        import densecore_amd as dc
        return list(dc.moe_route(st["x"], top, scoring=case["scoring"], bias=st["bias"], n_group=groups,
                                 topk_group=case["top_groups"], group_best=case["group_best"], renorm=True, scale=1.5,
                                 ids=st["ids"], weights=st["weights"]))
    x = st["x"].double()  # 64 bits: the order of scores next to each other
    if case["scoring"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score if st["bias"] is None else score + st["bias"].double()
    if groups > 1:
        by_group = choice.view(len(x), groups, -1)
        worth = torch.sort(by_group, dim=2, descending=True).values[:, :, :case["group_best"]].sum(2)
        best = torch.sort(worth, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        out = torch.ones_like(worth, dtype=torch.bool).scatter_(1, best, False)
        choice = torch.where(out[:, :, None], -math.inf, by_group).view(x.shape)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :top]
    got = torch.gather(score, 1, ids)
    return [ids.int(), (1.5 * got / got.sum(1, keepdim=True)).float()]


def _expert_products(x, w, scales, slots):
    """fp32 rows x [S, K] times the weights int8 [E, N, K] of each row's expert (slots [S]; E: none) and their scales -> [S, N]."""
    n_expert, n, _ = w.shape
    if len(slots) <= 64:  # a few rows: each one's weights by themselves
        e = slots.clamp(max=n_expert - 1)
        y = torch.bmm(w[e].float(), x[:, :, None]).view(len(slots), n) * scales[e]
    else:  # rows sorted by expert, every expert's padded to the most that one has
        order = torch.sort(slots, stable=True).indices
        counts = torch.bincount(slots, minlength=n_expert + 1)
        at = torch.arange(len(slots), device=DEV) - (torch.cumsum(counts, 0) - counts)[slots[order]]
        place = torch.empty_like(slots).scatter_(0, order, at)
        room = int(counts[:n_expert].max())
        ours = slots < n_expert
        rows = torch.zeros((n_expert, room, x.shape[1]), device=DEV)
        rows[slots[ours], place[ours]] = x[ours]
        full = torch.bmm(rows, w.float().transpose(1, 2)) * scales[:, None]
        y = full[slots.clamp(max=n_expert - 1), place.clamp(max=room - 1)]
    return torch.where((slots < n_expert)[:, None], y, 0.0)


def _slots(ids, n_expert):
    flat = ids.view(-1).long()
    return torch.where((flat >= 0) & (flat < n_expert), flat, n_expert)


def _run_up(st):
    case = st["case"]
    if own:
        import densecore_amd as dc
        plan = dc.moe_plan(st["ids"], case["experts"], plan=st["plan"])
        return dc.moe_gate_up_i8(plan, st["wg"], st["wgs"], st["wu"], st["wus"], st["x"], st["xs"], case["top"], h=st["h"])
    slots = _slots(st["ids"], case["experts"])
    x = (st["x"].float() * st["xs"][:, None]).repeat_interleave(case["top"], 0)
    gate = _expert_products(x, st["wg"], st["wgs"], slots)
    return gate / (1.0 + torch.exp(-gate)) * _expert_products(x, st["wu"], st["wus"], slots)


def _run_down(st):
    case = st["case"]
    if own:
        import densecore_amd as dc
        plan = dc.moe_plan(st["ids"], case["experts"], plan=st["plan"])
        return dc.moe_down_i8(plan, st["w"], st["ws"], st["h"], st["hs"], st["weights"], r=st["r"], y=st["y"],
                              workspace=st["ws_mem"])
    y = _expert_products(st["h"].float() * st["hs"][:, None], st["w"], st["ws"], _slots(st["ids"], case["experts"]))
    y = (y.view(-1, case["top"], case["n"]) * st["weights"][:, :, None]).sum(1)
    return y if st["r"] is None else y + st["r"]


def run(state):
    return {"norm": _run_norm, "product": _run_product, "route": _run_route, "up": _run_up, "down": _run_down}[
        state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _touched(case):
    """Experts that some token has, as expected of even choices."""
    e = case["experts"]
    return e * (1.0 - (1.0 - case["top"] / e) ** case["rows"])


def work(case):
    op, m = case["op"], case["rows"]
    size = 2 if "F16" in (case.get("dtype"), case.get("out")) else 4
    if op == "norm":
        k = case["width"]
        return {"bytes": m * k * (size + 1 + (8 if case["residual"] else 0)) + 4 * (m + k), "flops": 6 * m * k}
    if op == "route":
        return {"bytes": m * case["experts"] * size + 8 * m * case["top"], "flops": 8 * m * case["experts"]}
    n, k = case["n"], case["k"]
    if op == "product":
        add = {"none": 0, "residual": 4 * m * n, "bias": 4 * n}[case["add"]]
        return {"bytes": n * k + m * k + 4 * (n + m) + m * n * size + add, "flops": 2 * m * n * k}
    all_rows, slots, experts = m + case["pad"], m * case["top"], _touched(case)
    if op == "up":
        return {"bytes": int(2 * experts * n * (k + 4) + m * (k + 4) + all_rows * case["top"] * (4 * n + 4)),
                "flops": 4 * slots * n * k}
    return {"bytes": int(experts * n * (k + 4) + slots * (k + 8) + all_rows * case["top"] * 4
                         + 4 * all_rows * n * (2 if case["residual"] else 1)), "flops": 2 * slots * n * k}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_norm(case, st):
    h = st["x"].to(torch.float64)
    if case["residual"]:
        h = h + st["r"].to(torch.float64)
    kept = h.to(torch.float32).to(torch.float64)  # the residual stream is kept in 32 bits
    y = kept * st["w"].to(torch.float64)
    rms = torch.linalg.vector_norm(kept, dim=1) / math.sqrt(case["width"])
    y = y / torch.sqrt(rms ** 2 + EPS)[:, None]
    step = y.abs().max(dim=1).values / 127
    return [torch.round(y / step[:, None]) * step[:, None], step] + ([h] if case["residual"] else [])


def _exact_product(case, st):
    y = (st["x"].to(torch.float64) * st["xs"].to(torch.float64)[:, None]) @ st["w"].to(torch.float64).T
    y *= st["ws"].to(torch.float64)
    return y if st["r"] is None else y + st["r"].to(torch.float64)


def _exact_route(case, st):
    x = st["x"].to(torch.float64)
    score = torch.softmax(x, 1) if case["scoring"] == "softmax" else torch.sigmoid(x)
    choice = score if st["bias"] is None else score + st["bias"].to(torch.float64)
    if case["groups"] > 1:
        per = case["experts"] // case["groups"]
        parts = choice.split(per, 1)
        worth = torch.stack([torch.topk(p, min(case["group_best"], per), dim=1).values.sum(1) for p in parts], 1)
        keep = torch.topk(worth, case["top_groups"], dim=1).indices
        allowed = torch.zeros(worth.shape, dtype=torch.bool, device=DEV).scatter_(1, keep, True)
        choice = choice.masked_fill(~allowed.repeat_interleave(per, 1), -math.inf)
    got = score.gather(1, torch.topk(choice, case["top"], dim=1).indices)
    return [None, 1.5 * got / got.sum(1, keepdim=True)]


def _exact_experts(ids, n_expert, rows, matrices):
    """For each expert's slots: the products of `rows` (float64 [slots, K]) with each (weights, scales), in place of no slot zeros."""
    flat = ids.reshape(-1).long()
    outs = [torch.zeros((len(flat), w.shape[1]), dtype=torch.float64, device=DEV) for w, _ in matrices]
    for e in range(n_expert):
        mine = (flat == e).nonzero()[:, 0]
        if len(mine):
            for out, (w, s) in zip(outs, matrices):
                out[mine] = rows[mine] @ (w[e].to(torch.float64) * s[e].to(torch.float64)[:, None]).T
    return outs


def _exact_up(case, st):
    x = st["x"].to(torch.float64) * st["xs"].to(torch.float64)[:, None]
    token = torch.arange(st["ids"].numel(), device=DEV) // case["top"]
    gate, up = _exact_experts(st["ids"], case["experts"], x[token], [(st["wg"], st["wgs"]), (st["wu"], st["wus"])])
    return gate * torch.sigmoid(gate) * up


def _exact_down(case, st):
    h = st["h"].to(torch.float64) * st["hs"].to(torch.float64)[:, None]
    (y,) = _exact_experts(st["ids"], case["experts"], h, [(st["w"], st["ws"])])
    y = torch.einsum("mjn,mj->mn", y.view(*st["ids"].shape, case["n"]), st["weights"].to(torch.float64))
    return y if st["r"] is None else y + st["r"].to(torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "product": _exact_product, "route": _exact_route, "up": _exact_up, "down": _exact_down}[
        case["op"]](case, st)
