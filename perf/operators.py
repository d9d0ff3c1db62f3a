"""The mixture-of-experts operators on 4-bit weights, as cases that can be timed and compared.

A case is a dict with an ``op`` and its sizes and options.  ``M`` tokens, ``E`` experts, ``k`` of them for each token:

``route``    scores of every token against every expert -> the ``k`` experts of each token and their weights.
``up``       the experts' first product: every token times the gate and up rows of each of its experts, silu(gate) * up.
``down``     the experts' second product: the k results of a token, weighted and added up.
``layer``    the three together, as a program runs them between two residual additions.

Weights are those of w4a16_gemm: packed uint4 (low nibble first), a scale and a zero point for each group along K, and
dequantised W = T(T(u - z) * s) with T the activations' type.  That is what a weight IS in this package (dequantize_w4 gives
the same bits), so the plain form and exact() round it the same way; what is computed from it they do not round before
the end of each operator.
"""
import functools

import torch

own = False

_T = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# the most that a case may cost: the products and the weights of the listed ones that have most of them
_MOST_PRODUCTS = 8192 * 8 * 2 * 1024 * 2048
_MOST_WEIGHTS = 256 * 3 * 1024 * 4096


def listed():
    return [
        # the smallest call: the router's scores of the one token that is being decoded
        {"name": "route token", "op": "route", "M": 1, "E": 64, "k": 6, "scoring": "softmax", "groups": 1, "kept": 1, "bias": False, "renormalize": True, "dtype": "float32"},
        # a decode batch of a router without groups, scores straight out of a 16-bit product
        {"name": "route batch", "op": "route", "M": 259, "E": 128, "k": 8, "scoring": "softmax", "groups": 1, "kept": 1, "bias": False, "renormalize": True, "dtype": "bfloat16"},
        # prefill through a router with a bias for balance and groups of experts: the longest listed
        {"name": "route prefill", "op": "route", "M": 8192, "E": 256, "k": 8, "scoring": "sigmoid", "groups": 8, "kept": 4, "bias": True, "renormalize": True, "dtype": "float32"},
        # one token against the gate and up rows of its six experts
        {"name": "up token", "op": "up", "M": 1, "E": 64, "k": 6, "N": 1408, "K": 2048, "group": 128, "dtype": "float16", "zeros": "tensor", "share": 1.0},
        # a decode batch that meets most of many small experts
        {"name": "up batch", "op": "up", "M": 48, "E": 128, "k": 8, "N": 768, "K": 2048, "group": 128, "dtype": "bfloat16", "zeros": "scalar", "share": 1.0},
        # a prompt of an odd length against a few experts of a large projection
        {"name": "up prompt", "op": "up", "M": 211, "E": 8, "k": 2, "N": 14336, "K": 4096, "group": 64, "dtype": "float16", "zeros": "tensor", "share": 1.0},
        # prefill: the most products
        {"name": "up prefill", "op": "up", "M": 8192, "E": 64, "k": 8, "N": 1024, "K": 2048, "group": 128, "dtype": "bfloat16", "zeros": "scalar", "share": 1.0},
        # one token against the down rows of two large experts
        {"name": "down token", "op": "down", "M": 1, "E": 8, "k": 2, "N": 4096, "K": 14336, "group": 64, "dtype": "float16", "zeros": "tensor", "share": 1.0},
        # a decode batch on one of several GPUs: half of the chosen experts are elsewhere (their slots hold -1)
        {"name": "down batch", "op": "down", "M": 96, "E": 64, "k": 8, "N": 2048, "K": 768, "group": 128, "dtype": "bfloat16", "zeros": "scalar", "share": 0.5},
        # prefill of an odd number of tokens, rows with eleven groups
        {"name": "down prefill", "op": "down", "M": 4099, "E": 64, "k": 6, "N": 2048, "K": 1408, "group": 128, "dtype": "float16", "zeros": "tensor", "share": 1.0},
        # a decode step of sixteen sequences through a layer of many experts
        {"name": "layer batch", "op": "layer", "M": 16, "E": 256, "k": 8, "N": 1024, "K": 4096, "group": 128, "dtype": "bfloat16", "zeros": "tensor", "share": 1.0,
         "scoring": "sigmoid", "groups": 8, "kept": 4, "bias": True, "renormalize": True},
        # a chunk of prompts through a layer of a few experts
        {"name": "layer prefill", "op": "layer", "M": 2048, "E": 16, "k": 2, "N": 2048, "K": 4096, "group": 128, "dtype": "float16", "zeros": "scalar", "share": 1.0,
         "scoring": "softmax", "groups": 1, "kept": 1, "bias": False, "renormalize": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "up", "up", "down", "down", "layer"])
    while True:
        E = rng.choice([8, 16, 32, 60, 64, 128, 160, 256])
        c = {"op": op, "M": _log(rng, 1, 8192), "E": E, "k": rng.randint(1, 8)}
        if op in ("route", "layer"):
            groups = rng.choice([g for g in (1, 1, 4, 8) if E % g == 0 and E // g >= 8])
            kept = groups if groups == 1 else rng.randint(groups // 2, groups - 1)
            c.update(scoring=rng.choice(["softmax", "sigmoid"]), groups=groups, kept=kept, bias=rng.random() < 0.5, renormalize=rng.random() < 0.75)
        if op == "route":
            return {**c, "dtype": rng.choice(["float32", "float16", "bfloat16"])}
        c.update(N=64 * _log(rng, 4, 224), K=64 * _log(rng, 4, 224), dtype=rng.choice(["float16", "bfloat16"]), zeros=rng.choice(["tensor", "scalar"]), share=1.0)
        c["group"] = rng.choice([g for g in (32, 64, 128, 128) if c["K"] % g == 0 and (op != "layer" or c["N"] % g == 0)])
        if op != "layer":
            c["share"] = rng.choice([1.0, 1.0, 0.5])
        of_expert = {"up": 2, "down": 1, "layer": 3}[op] * c["N"] * c["K"]
        if E * of_expert <= _MOST_WEIGHTS and c["M"] * c["k"] * of_expert <= _MOST_PRODUCTS:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, M, E, k = case["op"], case["M"], case["E"], case["k"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    def weights(N, K, dtype):
        G = K // case["group"]
        words = torch.randint(-(2**63), 2**63 - 1, (E, N, K // 16), generator=g, device="cuda", dtype=torch.int64)
        zeros = torch.randint(6, 10, (E, N, G), generator=g, device="cuda").to(dtype) if case["zeros"] == "tensor" else 8
        return words.view(torch.uint8), uniform(0.005, 0.02, E, N, G).to(dtype), zeros

    s = {"case": case}
    if op in ("route", "layer"):
        # some experts are asked for more often than others; the bias that balances them takes part of that back
        favour = normal(E)
        s["logits"] = (normal(M, E) * 1.5 + favour).to(_T[case["dtype"]] if op == "route" else torch.float32)
        s["bias"] = -0.05 * favour if case["bias"] else None
    if op != "route":
        N, K, dtype = case["N"], case["K"], _T[case["dtype"]]
        if op == "down":
            # what silu(gate) * up of the first product looks like: small values and a few large ones
            gate, up = normal(M, k, K) * 2, normal(M, k, K) * 2
            s["hidden"] = (gate * torch.sigmoid(gate) * up).to(dtype)
            s["down"] = weights(N, K, dtype)
        else:
            s["x"] = normal(M, K).to(dtype)
            s["up"] = weights(2 * N, K, dtype)
        if op == "layer":
            s["down"] = weights(K, N, dtype)
        else:
            everywhere = max(k, round(E / case["share"]))
            score, ids = (normal(M, everywhere) + 0.7 * normal(everywhere)).topk(k, dim=1)
            s["ids"] = torch.where(ids < E, ids, -1).to(torch.int32)
            s["weights"] = torch.softmax(score, dim=1)
    return s


# ---- the framework's operators -----------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kernels(op, E, k, N, K, group, dtype, zeros, scoring, groups, kept, bias, renormalize):
    """The kernel objects that a program makes once: they take any number of tokens."""
    from tilelang_ascend_amd import ops

    z = "tensor" if zeros == "tensor" else 8
    route = up = down = None
    if op in ("route", "layer"):
        route = ops.moe_route(E, k, scoring=scoring, n_group=groups, topk_group=kept, renormalize=renormalize, with_bias=bias,
                              in_dtype=dtype if op == "route" else "float32")
    if op in ("up", "layer"):
        up = ops.moe_gate_up_w4a16(E, k, N, K, group_size=group, in_dtype=dtype, zeros=z)
    if op == "down":
        down = ops.moe_down_w4a16(E, k, N, K, group_size=group, in_dtype=dtype, out_dtype=dtype, zeros=z)
    if op == "layer":
        down = ops.moe_down_w4a16(E, k, K, N, group_size=group, in_dtype=dtype, out_dtype=dtype, zeros=z)
    return route, up, down


def _run_own(s):
    c = s["case"]
    route, up, down = _kernels(c["op"], c["E"], c["k"], c.get("N"), c.get("K"), c.get("group"), c["dtype"], c.get("zeros"), c.get("scoring"),
                               c.get("groups"), c.get("kept"), c.get("bias"), c.get("renormalize"))

    def of(w):
        return w if isinstance(w[2], torch.Tensor) else w[:2]

    if route is not None:
        weights, ids = route(s["logits"], s["bias"]) if c["bias"] else route(s["logits"])
        if c["op"] == "route":
            return weights, ids
    else:
        weights, ids = s["weights"], s["ids"]
    if c["op"] == "up":
        return up(s["x"], ids, *of(s["up"]))
    if c["op"] == "down":
        return down(s["hidden"], ids, weights, *of(s["down"]))
    return weights, ids, down(up(s["x"], ids, *of(s["up"])), ids, weights, *of(s["down"]))


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _plain_route(logits, bias, c):
    # in 64 bits: which of two near scores is larger decides an expert
    x = logits.double()
    if c["scoring"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if bias is None else score + bias.double()
    if c["groups"] > 1:
        M, E = x.shape
        best = choice.view(M, c["groups"], -1).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, : c["kept"]]
        is_kept = (kept[:, :, None] == torch.arange(E, device=x.device)[None, None] // (E // c["groups"])).any(1)
        choice = torch.where(is_kept, choice, float("-inf"))
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, : c["k"]]
    weights = score.gather(1, ids)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return weights.float(), ids.to(torch.int32)


def _plain_dequantized(packed, scales, zeros):
    """[E, N, K] in 32 bits, of packed [E, N, K / 2]; each of the two operations rounded to the scales' type."""
    E, N, G = scales.shape
    u = torch.stack((packed & 15, packed >> 4), 3).view(E, N, G, -1).to(scales.dtype)
    z = zeros[..., None] if isinstance(zeros, torch.Tensor) else zeros
    return ((u - z) * scales[..., None]).view(E, N, -1).float()


def _plain_product(rows, ids, w):
    """rows [P, K] times the weights of expert ids[p]: [P, N] in 32 bits, 0 where there is no expert."""
    E = w[0].shape[0]
    x, ids = rows.float(), ids.long()
    live = ids >= 0
    if ids.numel() <= E:
        at = ids.clamp(min=0)
        own_w = _plain_dequantized(w[0][at], w[1][at], w[2][at] if isinstance(w[2], torch.Tensor) else w[2])
        y = torch.bmm(own_w, x[:, :, None])[:, :, 0]
    else:
        key, order = torch.where(live, ids, E).sort(stable=True)
        count = torch.bincount(key, minlength=E + 1)
        place = torch.arange(len(key), device=x.device) - (count.cumsum(0) - count)[key]
        most = max(1, int(count[:E].max()))
        table = x.new_zeros(E + 1, most, x.shape[1])
        mine = key < E
        table[key[mine], place[mine]] = x[order[mine]]
        y = torch.bmm(table[:E], _plain_dequantized(*w).transpose(1, 2))[key.clamp(max=E - 1), place.clamp(max=most - 1)]
        y = torch.empty_like(y).index_copy_(0, order, y)
    return torch.where(live[:, None], y, 0.0)


def _plain_up(x, ids, w):
    M, k = ids.shape
    y = _plain_product(x.repeat_interleave(k, 0), ids.reshape(-1), w)
    gate, up = y.chunk(2, 1)
    return (gate / (1 + torch.exp(-gate)) * up).view(M, k, -1).to(x.dtype)


def _plain_down(hidden, ids, weights, w):
    M, k, K = hidden.shape
    y = _plain_product(hidden.view(M * k, K), ids.reshape(-1), w).view(M, k, -1)
    return (y * weights[:, :, None]).sum(1).to(hidden.dtype)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "up":
        return _plain_up(s["x"], s["ids"], s["up"])
    if c["op"] == "down":
        return _plain_down(s["hidden"], s["ids"], s["weights"], s["down"])
    weights, ids = _plain_route(s["logits"], s["bias"], c)
    if c["op"] == "route":
        return weights, ids
    return weights, ids, _plain_down(_plain_up(s["x"], ids, s["up"]), ids, weights, s["down"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what the operators cannot do without ------------------------------------------------------------------------------
def work(case):
    op, M, E, k = case["op"], case["M"], case["E"], case["k"]
    moved = flops = 0
    if op in ("route", "layer"):
        moved += M * E * (4 if op == "layer" or case["dtype"] == "float32" else 2) + (4 * E if case["bias"] else 0) + 8 * M * k
        flops += 4 * M * E
    if op == "route":
        return {"bytes": moved, "flops": flops}
    N, K, share = case["N"], case["K"], case["share"]
    # the experts that some token asks for, were all asked for alike
    met = E * (1 - (1 - share * k / E) ** M)
    of_row = {n: n / 2 + n / case["group"] * (4 if case["zeros"] == "tensor" else 2) for n in (K, N)}
    pairs = M * k * share
    if op in ("up", "layer"):
        moved += met * 2 * N * of_row[K] + 2 * M * K + 4 * M * k + (2 * M * k * N if op == "up" else 0)
        flops += 2 * pairs * 2 * N * K
    if op == "down":
        moved += met * N * of_row[K] + 2 * pairs * K + 8 * M * k + 2 * M * N
        flops += 2 * pairs * N * K
    if op == "layer":
        moved += met * K * of_row[N] + 2 * M * K
        flops += 2 * pairs * N * K
    return {"bytes": int(moved), "flops": int(flops)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_route(s, c):
    x = s["logits"].to(torch.float64)
    if c["scoring"] == "softmax":
        p = (x - torch.logsumexp(x, 1, keepdim=True)).exp()
    else:
        p = torch.where(x >= 0, 1 / (1 + (-x).exp()), x.exp() / (1 + x.exp()))
    v = p if s["bias"] is None else p + s["bias"].to(torch.float64)
    if c["groups"] > 1:
        per = x.shape[1] // c["groups"]
        of_group = torch.stack([t.topk(2, dim=1).values.sum(1) for t in v.split(per, 1)], 1)
        barred = torch.argsort(of_group, dim=1, descending=True, stable=True)[:, c["kept"]:]
        for i in range(barred.shape[1]):
            cols = barred[:, i: i + 1] * per + torch.arange(per, device=x.device)
            v = v.scatter(1, cols, -torch.inf)
    ids = torch.argsort(v, dim=1, descending=True, stable=True)[:, : c["k"]]
    w = torch.take_along_dim(p, ids, 1)
    return (w / w.sum(1, keepdim=True) if c["renormalize"] else w), ids


def _exact_matrix(w, e):
    packed, scales, zeros = w
    T, K = scales.dtype, packed.shape[2] * 2
    u = torch.empty(packed.shape[1], K, dtype=torch.float64, device=packed.device)
    u[:, 0::2] = packed[e] % 16
    u[:, 1::2] = packed[e] // 16
    spread = K // scales.shape[2]
    z = zeros[e].to(torch.float64).repeat_interleave(spread, 1) if torch.is_tensor(zeros) else float(zeros)
    return ((u - z).to(T).to(torch.float64) * scales[e].to(torch.float64).repeat_interleave(spread, 1)).to(T).to(torch.float64)


def _exact_product(rows, ids, w, per_token):
    """Entry [t, j]: the row of token t (of slot j where `per_token` is false) times the matrix of its expert."""
    M, k = ids.shape
    y = torch.zeros(M, k, w[0].shape[1], dtype=torch.float64, device=rows.device)
    for e in torch.unique(ids).tolist():
        if e >= 0:
            t, j = torch.nonzero(ids == e, as_tuple=True)
            y[t, j] = (rows[t] if per_token else rows[t, j]).to(torch.float64) @ _exact_matrix(w, e).T
    return y


def _exact_up(s, ids):
    a, b = _exact_product(s["x"], ids, s["up"], True).tensor_split(2, 2)
    return a * torch.sigmoid(a) * b


def _exact_down(hidden, s, ids, weights):
    return torch.bmm(weights.to(torch.float64)[:, None], _exact_product(hidden, ids, s["down"], False))[:, 0]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "up":
        return _exact_up(s, s["ids"])
    if case["op"] == "down":
        return _exact_down(s["hidden"], s, s["ids"], s["weights"])
    weights, ids = _exact_route(s, case)
    if case["op"] == "route":
        return weights, ids
    # what one operator hands to the next has its type: the weights 32 bits, the hidden rows the activations'
    hidden = _exact_up(s, ids).to(s["x"].dtype)
    return weights, ids, _exact_down(hidden, s, ids, weights.float())
