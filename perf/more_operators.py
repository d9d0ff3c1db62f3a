"""The operators around and beside the quantised projections of a transformer block, as cases that can be timed and compared.

A case is a dict with an ``op``, its number of tokens ``M``, its sizes and options:

``norm``    the residual's addition and the root-mean-square norm: N values a token.
``gated``   silu(gate) * up of N gates and N ups a token, between the two products of an MLP.
``update``  the low-rank adapters of many requests beside a projection from K to N values, which may be up to three side by side
            (``N1`` and ``N2``, 0: none): every token's own adapter of L, or none.

``out`` of the first two: "float" the activations' type, "int8" codes with a scale for each token (what the int8 products take), "both".
Codes are returned as the values that they stand for, code * scale, in the activations' type: a product of torch's that is part of the pass
on either side.
"""
import functools

import torch

own = False

_T = {"float16": torch.float16, "bfloat16": torch.bfloat16}
# the most that a drawn case may cost: what the largest listed ones move, and their dense plain form multiplies
_MOST_NORM, _MOST_GATED, _MOST_ROWS, _MOST_PRODUCTS, _MOST_WEIGHTS = 8192 * 8192, 8192 * 14336, 8192 * (4096 + 2 * 14336), 8192 * 16 * 32 * (4096 + 14336), 1 << 28


def listed():
    return [
        # the smallest call: the norm ahead of a projection of the one token that is being decoded
        {"name": "norm token", "op": "norm", "M": 1, "N": 4096, "residual": True, "out": "float", "eps": 1e-6, "dtype": "bfloat16"},
        # a decode batch ahead of an int8 projection
        {"name": "norm batch", "op": "norm", "M": 48, "N": 5120, "residual": True, "out": "int8", "eps": 1e-5, "dtype": "float16"},
        # a prompt of an odd length ahead of an int8 projection with adapters, which take the 16-bit values
        {"name": "norm prompt", "op": "norm", "M": 1021, "N": 3584, "residual": True, "out": "both", "eps": 1e-6, "dtype": "bfloat16"},
        # prefill ahead of a 4-bit projection
        {"name": "norm prefill", "op": "norm", "M": 8192, "N": 8192, "residual": True, "out": "float", "eps": 1e-5, "dtype": "bfloat16"},
        # one token between the products of an MLP
        {"name": "gated token", "op": "gated", "M": 1, "N": 11008, "out": "float", "dtype": "float16"},
        # a decode batch ahead of an int8 projection
        {"name": "gated batch", "op": "gated", "M": 67, "N": 14336, "out": "int8", "dtype": "bfloat16"},
        # prefill ahead of a 4-bit projection
        {"name": "gated prefill", "op": "gated", "M": 8192, "N": 14336, "out": "float", "dtype": "bfloat16"},
        # one token of a request that has an adapter
        {"name": "update token", "op": "update", "M": 1, "L": 8, "rank": 16, "K": 4096, "N": 4096, "N1": 0, "N2": 0, "prompts": 0, "share": 1.0, "dtype": "float16"},
        # a decode batch beside the product for queries, keys and values: most requests have an adapter of their own, some have none
        {"name": "update batch", "op": "update", "M": 64, "L": 48, "rank": 16, "K": 4096, "N": 4096, "N1": 1024, "N2": 1024, "prompts": 0, "share": 0.8, "dtype": "bfloat16"},
        # a large decode batch on fewer adapters of a high rank, beside gate and up
        {"name": "update wide batch", "op": "update", "M": 259, "L": 32, "rank": 64, "K": 4096, "N": 11008, "N1": 11008, "N2": 0, "prompts": 0, "share": 0.9, "dtype": "float16"},
        # a chunk of two prompts with the tokens that are being decoded behind it, beside the down product
        {"name": "update prompt", "op": "update", "M": 1003, "L": 12, "rank": 8, "K": 11008, "N": 4096, "N1": 0, "N2": 0, "prompts": 2, "share": 0.8, "dtype": "float16"},
        # prefill of several prompts
        {"name": "update prefill", "op": "update", "M": 8192, "L": 16, "rank": 32, "K": 4096, "N": 14336, "N1": 0, "N2": 0, "prompts": 9, "share": 0.9, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "gated", "update", "update"])
    while True:
        c = {"op": op, "M": _log(rng, 1, 8192), "dtype": rng.choice(["float16", "bfloat16"])}
        if op in ("norm", "gated"):
            # widths are multiples of eight but for a few odd ones
            c["N"] = 8 * _log(rng, 64, 2048) - (rng.randint(1, 7) if rng.random() < 0.1 else 0)
            c["out"] = rng.choice(["float", "int8", "both"])
            if op == "norm":
                c.update(residual=rng.random() < 0.75, eps=rng.choice([1e-6, 1e-5]))
            if c["M"] * c["N"] <= (_MOST_NORM if op == "norm" else _MOST_GATED):
                return c
            continue
        c.update(L=_log(rng, 1, 128), rank=rng.choice([8, 16, 16, 32, 64]), K=32 * _log(rng, 16, 448), N=16 * _log(rng, 32, 896), N1=0, N2=0, prompts=0, share=rng.choice([1.0, 0.9, 0.5]))
        parts = rng.choice([1, 1, 2, 3])
        if parts > 1:
            c["N1"] = c["N"] if parts == 2 else 16 * max(1, c["N"] // 64)
        if parts > 2:
            c["N2"] = c["N1"]
        if c["M"] > 256:
            c["prompts"] = rng.randint(1, 12)
        of_adapter = c["rank"] * (parts * c["K"] + c["N"] + c["N1"] + c["N2"])
        if (c["M"] * (c["K"] + 2 * (c["N"] + c["N1"] + c["N2"])) <= _MOST_ROWS and c["M"] * c["L"] * of_adapter <= _MOST_PRODUCTS
                and c["L"] * of_adapter <= _MOST_WEIGHTS):
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _widths(case):
    return [n for n in (case["N"], case["N1"], case["N2"]) if n]


def _decoded(case):
    """How many of an update's tokens are those of requests that are being decoded."""
    return case["M"] if not case["prompts"] else min(64, case["M"] // 32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, N, dtype = case["M"], case["N"], _T[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "norm":
        # the residual stream has a few channels that are much larger than the others
        loud = 1 + 30 * (torch.rand(N, generator=g, device="cuda") < 0.004)
        s["x"] = normal(M, N).to(dtype)
        s["residual"] = (normal(M, N) * 3 * loud).to(dtype) if case["residual"] else None
        s["weight"] = (0.6 + 0.2 * normal(N)).to(dtype)
    elif case["op"] == "gated":
        s["x"] = (normal(M, 2 * N) * 2).to(dtype)
    else:
        L, r, K, widths, decoded = case["L"], case["rank"], case["K"], _widths(case), _decoded(case)
        s["x"] = normal(M, K).to(dtype)
        s["y"] = (normal(M, sum(widths)) * 2).to(dtype)
        s["a"] = (normal(L, len(widths) * r, K) * K**-0.5).to(dtype)
        s["b"] = (normal(L, sum(widths), r) * 0.2).to(dtype)
        s["scaling"] = torch.rand(L, generator=g, device="cuda") * 2 + 0.5
        # requests: one for each decoded token, behind the prompts
        request = torch.arange(M, device="cuda")
        if case["prompts"]:
            cuts = torch.randint(0, M, (case["prompts"] - 1,), generator=g, device="cuda").sort().values
            request = torch.where(request < M - decoded, torch.searchsorted(cuts, request, right=True), request)
        adapter = torch.randint(0, L, (M,), generator=g, device="cuda")
        adapter = torch.where(torch.rand(M, generator=g, device="cuda") < case["share"], adapter, -1)
        s["ids"] = adapter[request].to(torch.int32)
    return s


# ---- the framework's operators -----------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kernel(op, N, out, residual, eps, dtype, L, rank, K, N1, N2):
    """The kernel object that a program makes once: it takes any number of tokens."""
    from tilelang_ascend_amd import ops

    if op == "norm":
        return ops.residual_rms_norm(N, eps=eps, outputs=out, with_residual=residual, in_dtype=dtype)
    if op == "gated":
        return ops.gated_silu(N, outputs=out, in_dtype=dtype)
    return ops.low_rank_update(L, rank, tuple(n for n in (N, N1, N2) if n), K, in_dtype=dtype, out_dtype=dtype)


def _run_own(s):
    c = s["case"]
    kernel = _kernel(c["op"], c["N"], c.get("out"), c.get("residual"), c.get("eps"), c["dtype"], c.get("L"), c.get("rank"), c.get("K"), c.get("N1"), c.get("N2"))
    if c["op"] == "update":
        return kernel(s["x"], s["y"], s["ids"], s["a"], s["b"], s["scaling"])
    if c["op"] == "gated":
        got = kernel(s["x"])
    elif c["residual"]:
        got = kernel(s["x"], s["residual"], s["weight"])
    else:
        got = kernel(s["x"], s["weight"])
    if c["out"] == "float":
        return got
    *others, codes, scales = got
    return [*others, torch.mul(codes, scales[:, None], out=torch.empty(codes.shape, dtype=_T[c["dtype"]], device=codes.device)), scales]


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _plain_outputs(y, c, dtype):
    """Of y in 64 or 32 bits: rounded to the activations' type, and / or as codes of 8 bits times their scales."""
    got = [y.to(dtype)] if c["out"] != "int8" else []
    if c["out"] != "float":
        scales = y.abs().amax(1, keepdim=True).clamp(min=1e-4) / 127
        codes = (y / scales).clamp(-127, 127).round()
        got += [(codes.float() * scales.float()).to(dtype), scales[:, 0].float()]
    return got if len(got) > 1 else got[0]


def _plain_norm(s, c):
    x = s["x"]
    h = (x.float() + s["residual"].float()).to(x.dtype) if c["residual"] else x
    # in 64 bits where codes are made: a value next to the middle of two of them
    z = h.double() if c["out"] != "float" else h.float()
    y = z / torch.sqrt((z * z).mean(1, keepdim=True) + c["eps"]) * s["weight"].to(z.dtype)
    got = _plain_outputs(y, c, x.dtype)
    if not c["residual"]:
        return got
    return [h, *got] if isinstance(got, list) else [h, got]


def _plain_gated(s, c):
    gate, up = s["x"].to(torch.float64 if c["out"] != "float" else torch.float32).chunk(2, 1)
    return _plain_outputs(gate / (1 + torch.exp(-gate)) * up, c, s["x"].dtype)


def _plain_update(s, c):
    x, ids, L, r, widths = s["x"].float(), s["ids"].long(), c["L"], c["rank"], _widths(c)
    M, P = len(ids), len(widths)
    a, b, live = s["a"].float(), s["b"].float(), ids >= 0
    at = ids.clamp(min=0)
    if M <= L:
        # each token's own matrices
        h = torch.bmm(a[at], x[:, :, None]).view(M, P, r)
        delta = torch.cat([torch.bmm(w, h[:, p, :, None])[:, :, 0] for p, w in enumerate(b[at].split(widths, 1))], 1)
    else:
        # every token against every adapter, with all but its own taken out between the two products
        mine = torch.arange(L, device=x.device)[None, :] == ids[:, None]
        h = (x @ a.view(L * P * r, -1).T).view(M, L, P, r) * mine[:, :, None, None]
        delta = torch.cat([h[:, :, p].reshape(M, L * r) @ w.transpose(1, 2).reshape(L * r, -1) for p, w in enumerate(b.split(widths, 1))], 1)
    delta = delta * s["scaling"][at][:, None]
    return (s["y"].float() + torch.where(live[:, None], delta, 0.0)).to(s["y"].dtype)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    return {"norm": _plain_norm, "gated": _plain_gated, "update": _plain_update}[c["op"]](state, c)


# ---- what the operators cannot do without ------------------------------------------------------------------------------
def work(case):
    M, N = case["M"], case["N"]
    if case["op"] == "update":
        widths, r, K = _widths(case), case["rank"], case["K"]
        requests = case["prompts"] + _decoded(case) if case["prompts"] else M
        met = case["L"] * (1 - (1 - case["share"] / case["L"]) ** requests)  # the adapters that some request has
        of_adapter = r * (len(widths) * K + sum(widths))
        rows = M * case["share"]
        return {"bytes": int(met * (2 * of_adapter + 4) + 2 * rows * K + 4 * M * sum(widths) + 4 * M), "flops": int(2 * rows * of_adapter)}
    codes, floats = case["out"] != "float", case["out"] != "int8"
    if case["op"] == "gated":
        return {"bytes": M * N * (4 + 2 * floats + codes) + 4 * M * codes, "flops": 8 * M * N}
    return {"bytes": M * N * (2 + 4 * case["residual"] + 2 * floats + codes) + 2 * N + 4 * M * codes, "flops": 6 * M * N}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_outputs(y, c, dtype):
    outs = []
    if c["out"] in ("float", "both"):
        outs.append(y)
    if c["out"] in ("int8", "both"):
        top = torch.linalg.vector_norm(y, ord=torch.inf, dim=1)
        scale = torch.maximum(top, torch.full_like(top, 1e-4)) / 127
        outs += [torch.round(y / scale.unsqueeze(1)) * scale.unsqueeze(1), scale]
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "norm":
        # the residual stream is held in the activations' type, and what is normalised is what it holds
        h = s["x"] if s["residual"] is None else torch.add(s["x"].to(f), s["residual"].to(f)).to(s["x"].dtype)
        z = h.to(f)
        length = torch.linalg.vector_norm(z, dim=1, keepdim=True)
        outs = _exact_outputs(torch.rsqrt(length.square() / z.shape[1] + case["eps"]) * z * s["weight"].to(f), case, h.dtype)
        if s["residual"] is not None:
            outs.insert(0, z)
    elif case["op"] == "gated":
        n = case["N"]
        z = s["x"].to(f)
        outs = _exact_outputs(z[:, :n] * torch.sigmoid(z[:, :n]) * z[:, n:], case, s["x"].dtype)
    else:
        out, r = s["y"].to(f), case["rank"]
        for adapter in torch.unique(s["ids"]).tolist():
            if adapter < 0:
                continue
            t = torch.nonzero(s["ids"] == adapter)[:, 0]
            h = s["x"][t].to(f) @ s["a"][adapter].to(f).T
            begin = 0
            for p, n in enumerate(_widths(case)):
                out[t, begin: begin + n] += s["scaling"][adapter].to(f) * (h[:, p * r: (p + 1) * r] @ s["b"][adapter, begin: begin + n].to(f).T)
                begin += n
        return out
    return outs if len(outs) > 1 else outs[0]
