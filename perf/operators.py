"""The expert-routing and 4-bit operators: what is measured, and their plain forms.

``own = False``: elementary torch operations in 32 bits, rounded once.
``own = True``: the calls a user of ``fack_b200`` makes.

A routed layer's state holds its plan as three plain tensors: ``row_of`` [T, k] (the sorted row of each token's
slot, -1 where it is not routed), ``src`` [T*k] (the pair t*k + j of each sorted row, -1 behind the last) and
``offsets`` [E + 1] (each expert's first row).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_GROUP = 128        # width of a quantisation group of the FP8 GEMM's activations
_QMAX = 240.0
_HBM_MOST = 2_200_000_000   # bytes of the largest drawn pass


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one token's choice of experts, as the router of a decode step gives it: launch latency
        {"name": "sort one token", "op": "sort", "tokens": 1, "topk": 8, "experts": 256, "of": 256, "ids": "int64"},
        # a long prefill on one of four expert-parallel ranks: three quarters of the pairs go elsewhere
        {"name": "sort prefill share", "op": "sort", "tokens": 65536, "topk": 8, "experts": 64, "of": 256, "ids": "int32"},
        # a small fp32 training step, an odd number of tokens, two of eight experts; output and gradient
        {"name": "gather train small", "op": "gather", "tokens": 1021, "topk": 2, "experts": 8, "of": 8, "dim": 2048, "type": "fp32", "grad": True},
        # a prefill-sized training step at the layer width 7168, eight rows a token; output and gradient
        {"name": "gather train wide", "op": "gather", "tokens": 8192, "topk": 8, "experts": 256, "of": 256, "dim": 7168, "type": "bf16", "grad": True},
        # the inputs of a decode batch's FP8 expert GEMMs
        {"name": "quantise decode", "op": "quant", "tokens": 16, "topk": 8, "experts": 256, "of": 256, "dim": 7168, "type": "bf16"},
        # the inputs of a prefill's FP8 expert GEMMs from an fp32 residual stream
        {"name": "quantise prefill", "op": "quant", "tokens": 4095, "topk": 4, "experts": 64, "of": 64, "dim": 7168, "type": "fp32"},
        # the end of a decode step's expert layer
        {"name": "combine decode", "op": "combine", "tokens": 8, "topk": 8, "experts": 256, "of": 256, "dim": 7168, "type": "bf16", "grad": False},
        # a training step's combine: output, and the gradients of the rows and of the routing weights
        {"name": "combine train", "op": "combine", "tokens": 4096, "topk": 6, "experts": 64, "of": 64, "dim": 4096, "type": "fp16", "grad": True},
        # one token through a projection of 7 MB
        {"name": "w4 one token", "op": "w4", "tokens": 1, "n": 7168, "k": 2048, "group": 128, "type": "bf16", "zeros": False},
        # a ragged batch through the widest layer, 235 MB, with zero points and small groups
        {"name": "w4 wide batch", "op": "w4", "tokens": 13, "n": 65536, "k": 7168, "group": 64, "type": "fp16", "zeros": True},
        # a decode step of two tokens: the experts' first product, which reads the tokens' own rows
        {"name": "experts first, 2 tokens", "op": "experts", "tokens": 2, "topk": 8, "experts": 64, "n": 4096, "k": 7168, "group": 128, "type": "bf16", "zeros": False, "sorted": False},
        # a decode batch's second product, which reads the sorted rows: most experts have a few
        {"name": "experts second, batch", "op": "experts", "tokens": 47, "topk": 6, "experts": 64, "n": 7168, "k": 2048, "group": 32, "type": "fp16", "zeros": True, "sorted": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "gather", "quant", "combine", "w4", "experts"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    topk = rng.randint(1, 8)
    experts = _log(rng, 8, 320)
    of = experts * rng.choice([1, 1, 1, 2, 4])
    if op == "sort":
        return {"op": op, "tokens": _log(rng, 1, 65536), "topk": topk, "experts": experts, "of": min(of, 512), "ids": rng.choice(["int64", "int32"])}
    if op in ("gather", "combine"):
        grad = rng.random() < 0.6
        dim = rng.choice([_log(rng, 65, 7168), 8 * _log(rng, 16, 896), 128 * rng.randint(4, 56)])
        most = _HBM_MOST // (dim * _BYTES[kind] * (topk * (3 if op == "combine" else 2) + 3))
        return {"op": op, "tokens": _log(rng, 1, max(1, min(8192, most))), "topk": topk, "experts": experts, "of": of, "dim": dim, "type": kind, "grad": grad}
    if op == "quant":
        kind = rng.choice(["bf16", "fp32"])
        return {"op": op, "tokens": _log(rng, 1, 8192), "topk": topk, "experts": experts, "of": of, "dim": 128 * rng.randint(1, 56), "type": kind}
    group = rng.choice([32, 64, 128])
    kind = rng.choice(["bf16", "fp16"])
    k = group * _log(rng, 256 // group, 7168 // group)
    n = 16 * _log(rng, 16, 512)
    if op == "w4":
        n = 16 * _log(rng, 16, 4096)
        return {"op": op, "tokens": _log(rng, 1, 32), "n": n, "k": k, "group": group, "type": kind, "zeros": rng.random() < 0.5}
    experts = _log(rng, 8, max(8, min(64, 1_800_000_000 // (n * k))))
    return {"op": op, "tokens": _log(rng, 1, 64), "topk": min(topk, experts), "experts": experts, "n": n, "k": k, "group": group, "type": kind,
            "zeros": rng.random() < 0.5, "sorted": rng.random() < 0.5}


def work(case):
    op, T = case["op"], case["tokens"]
    if op == "sort":
        pairs = T * case["topk"]
        return {"bytes": pairs * ((8 if case["ids"] == "int64" else 4) + 8) + 4 * (case["experts"] + 1), "flops": 0}
    if op in ("gather", "quant", "combine"):
        pairs, dim, es = T * case["topk"], case["dim"], _BYTES[case["type"]]
        routed = pairs * case["experts"] // case["of"]      # pairs that stay on this rank
        if op == "quant":
            return {"bytes": T * dim * es + pairs * (dim + dim // 32 + 4), "flops": 3 * T * dim}
        if op == "gather":
            back = routed * dim * es + T * dim * es + 4 * pairs if case["grad"] else 0
            return {"bytes": T * dim * es + pairs * dim * es + 4 * pairs + back, "flops": routed * dim if case["grad"] else 0}
        back = (routed + pairs + T) * dim * es + 12 * pairs if case["grad"] else 0
        return {"bytes": (routed + T) * dim * es + 8 * pairs + back, "flops": (5 if case["grad"] else 2) * routed * dim}
    n, k, groups = case["n"], case["k"], case["k"] // case["group"]
    weights = n * k / 2 + n * groups * (2 + (1 if case["zeros"] else 0))
    if op == "w4":
        return {"bytes": int(weights + 2 * T * (n + k)), "flops": 2 * T * n * k}
    rows = T * case["topk"]
    hit = case["experts"] * (1 - (1 - case["topk"] / case["experts"]) ** T)       # experts with a row, all alike
    return {"bytes": int(hit * weights + 2 * ((rows if case["sorted"] else T) * k + rows * n) + 8 * rows), "flops": 2 * rows * n * k}


# ----------------------------------------------------------------- inputs --

def _ids(g, T, topk, experts, of):
    """Router choices: the best of noisy logits over `of` experts, of which this rank holds `experts`."""
    logits = torch.randn((T, of), generator=g, device="cuda") + 0.5 * torch.randn((1, of), generator=g, device="cuda")
    top, ids = torch.topk(logits, topk, dim=1)
    return ids - (of - experts) // 2, torch.softmax(top, dim=1)


def _sorted_plan(ids, experts):
    flat = ids.reshape(-1).long()
    pairs = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=ids.device))
    rows = torch.arange(pairs, device=ids.device)
    routed = rows < offsets[experts]
    row_of = torch.empty_like(rows)
    row_of[order] = torch.where(routed, rows, -1)
    src = torch.where(routed, order, -1)
    return row_of.reshape(ids.shape).int(), src.int(), offsets.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, T = case["op"], case["tokens"]

    def randn(*shape, dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    state = {"case": case}
    if op != "w4":
        experts = case["experts"]
        ids, gates = _ids(g, T, case["topk"], experts, case.get("of", experts))
        if op == "sort":
            return {**state, "ids": ids.to(torch.int64 if case["ids"] == "int64" else torch.int32)}
        state["row_of"], state["src"], state["offsets"] = _sorted_plan(ids, experts)
        pairs = T * case["topk"]
    dtype = _TYPES[case["type"]]
    if op in ("gather", "quant"):
        state["x"] = randn(T, case["dim"], dtype=dtype)
        if op == "quant":       # a few large entries, as activations have
            state["x"] = torch.where(torch.rand(state["x"].shape, generator=g, device="cuda") < 1e-3, state["x"] * 50, state["x"])
        elif case["grad"]:
            state["dy"] = randn(pairs, case["dim"], dtype=dtype)
    elif op == "combine":
        state["y"], state["gates"] = randn(pairs, case["dim"], dtype=dtype), gates
        if case["grad"]:
            state["dout"] = randn(T, case["dim"], dtype=dtype)
    else:
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        lead = () if op == "w4" else (case["experts"],)
        state["w"] = torch.randint(0, 256, (*lead, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        state["scales"] = ((torch.rand((*lead, groups, n), generator=g, device="cuda") + 0.5) * 0.01).to(dtype)
        state["zeros"] = torch.randint(0, 16, (*lead, groups, n), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        state["x"] = randn(pairs if op == "experts" and case["sorted"] else T, k, dtype=dtype)
    return state


# -------------------------------------------------------------------- run --

def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    import fack_b200 as fb
    case = s["case"]
    op = case["op"]
    if op == "w4":
        return fb.gemv_w4(s["x"], s["w"], s["scales"], s["zeros"])
    if op == "sort":
        plan = fb.moe_sort(s["ids"], case["experts"])
        return plan.row_of, plan.src, plan.offsets
    plan = fb.MoePlan(s["row_of"], s["src"], s["offsets"])
    if op == "quant":
        return fb.moe_gather_quant(s["x"], plan)
    if op == "experts":
        return fb.gemv_w4_experts(s["x"], s["w"], s["scales"], plan, s["zeros"], sorted_rows=case["sorted"])
    if op == "gather":
        if not case["grad"]:
            return fb.moe_gather(s["x"], plan)
        x = s["x"].detach().requires_grad_()
        y = fb.moe_gather(x, plan)
        return y, torch.autograd.grad(y, x, s["dy"])[0]
    if not case["grad"]:
        return fb.moe_combine(s["y"], s["gates"], plan)
    y, gates = s["y"].detach().requires_grad_(), s["gates"].detach().requires_grad_()
    out = fb.moe_combine(y, gates, plan)
    dy, dgates = torch.autograd.grad(out, (y, gates), s["dout"])
    return out, dy, dgates


def _rows(values, index):
    """values[index], and zeros where the index is negative."""
    return values[index.clamp(min=0).long()].masked_fill_((index < 0).reshape(index.shape + (1,) * (values.dim() - 1)), 0)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "w4":
        return (s["x"].float() @ _weights(s["w"], s["scales"], s["zeros"], case["group"]).T).to(s["x"].dtype)
    if op == "sort":
        return _sorted_plan(s["ids"], case["experts"])
    row_of, src, topk = s["row_of"], s["src"], case["topk"]
    token = torch.where(src < 0, -1, src // topk)
    if op == "quant":
        groups = s["x"].float().reshape(case["tokens"], -1, _GROUP)
        scale = groups.abs().amax(dim=2) / _QMAX
        scale = torch.where(scale == 0, 1.0, scale)
        codes = (groups / scale[:, :, None]).clamp(-_QMAX, _QMAX).to(torch.float8_e4m3fn).reshape(s["x"].shape)
        xq = _rows(codes.view(torch.uint8), token).view(torch.float8_e4m3fn)
        return xq, scale[token.clamp(min=0).long()].masked_fill_((token < 0)[:, None], 1)
    if op == "gather":
        y = _rows(s["x"], token)
        if not case["grad"]:
            return y
        return y, _rows(s["dy"].float(), row_of).sum(dim=1).to(s["dy"].dtype)
    if op == "combine":
        picked = _rows(s["y"].float(), row_of)
        out = (s["gates"][:, :, None] * picked).sum(dim=1).to(s["y"].dtype)
        if not case["grad"]:
            return out
        dout = s["dout"].float()
        dgates = (dout[:, None, :] * picked).sum(dim=2)
        row_gate = _rows(s["gates"].reshape(-1, 1), src)
        return out, (row_gate * _rows(dout, token)).to(s["y"].dtype), dgates
    x = s["x"] if case["sorted"] else _rows(s["x"], token)
    return _experts(x.float(), s, case).to(s["x"].dtype)


def _weights(w, scales, zeros, group):
    """The 4-bit weights' values [..., N, K] in fp32."""
    codes = torch.stack((w & 15, w >> 4), dim=-1).flatten(-2).float()
    zero = 8.0 if zeros is None else zeros.float().transpose(-1, -2).repeat_interleave(group, dim=-1)
    return (codes - zero) * scales.float().transpose(-1, -2).repeat_interleave(group, dim=-1)


def _experts(x, s, case):
    rows, E = x.shape[0], case["experts"]
    r = torch.arange(rows, device=x.device)
    expert = torch.searchsorted(s["offsets"].long(), r, right=True) - 1
    routed = expert < E
    expert = expert.clamp(max=E - 1)
    zeros = s["zeros"]
    if rows < E:                            # few rows: each with its own expert's weights
        w = _weights(s["w"][expert], s["scales"][expert], None if zeros is None else zeros[expert], case["group"])
        y = torch.bmm(w, x[:, :, None])[:, :, 0]
    else:                                   # all experts, each with room for as many rows as it can have
        w = _weights(s["w"], s["scales"], zeros, case["group"])
        at = r - s["offsets"].long()[expert]
        padded = torch.zeros((E, case["tokens"], case["k"]), device=x.device)
        padded[expert, at] = x
        y = torch.bmm(padded, w.transpose(1, 2))[expert, at]
    return y.masked_fill_(~routed[:, None], 0)


# ------------------------------------------------------------------ exact --

def exact(case, seed):
    """run()'s outputs in 64 bits from the definitions; None in the place of whole numbers."""
    op = case["op"]
    if op == "sort":
        return None
    s = prepare(case, seed)
    topk = case.get("topk", 1)
    if op == "w4":
        return torch.cat([s["x"].double() @ _values(s["w"][i:i + 4096], s["scales"][:, i:i + 4096], None if s["zeros"] is None else s["zeros"][:, i:i + 4096], case["group"]).T
                          for i in range(0, case["n"], 4096)], dim=1)
    src = s["src"].tolist()
    count = len([p for p in src if p >= 0])                 # routed rows come first
    pair = s["src"][:count].long()
    owner = torch.div(pair, topk, rounding_mode="floor")
    if op == "quant":
        x = s["x"].double().reshape(case["tokens"], -1, _GROUP)
        scale = x.abs().max(dim=2).values / _QMAX
        scale[scale == 0] = 1
        q = (x / scale.unsqueeze(2)).reshape(case["tokens"], -1)
        xq = torch.zeros((len(src), case["dim"]), dtype=torch.float64, device="cuda")
        xs = torch.ones((len(src), case["dim"] // _GROUP), dtype=torch.float64, device="cuda")
        xq[:count], xs[:count] = q[owner], scale[owner]
        return xq, xs
    if op == "gather":
        y = torch.zeros((len(src), case["dim"]), dtype=torch.float64, device="cuda")
        y[:count] = s["x"].double()[owner]
        if not case["grad"]:
            return y
        dx = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        dx.index_add_(0, owner, s["dy"][:count].double())
        return y, dx
    if op == "combine":
        gate = s["gates"].double().reshape(-1)[pair].unsqueeze(1)
        y = s["y"][:count].double()
        out = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        out.index_add_(0, owner, gate * y)
        if not case["grad"]:
            return out
        d = s["dout"].double()[owner]
        dy = torch.zeros((len(src), case["dim"]), dtype=torch.float64, device="cuda")
        dy[:count] = gate * d
        dgates = torch.zeros(case["tokens"] * topk, dtype=torch.float64, device="cuda")
        dgates[pair] = torch.einsum("rd,rd->r", d, y)
        return out, dy, dgates.reshape(case["tokens"], topk)
    y = torch.zeros((len(src), case["n"]), dtype=torch.float64, device="cuda")
    bounds = s["offsets"].tolist()
    for e in range(case["experts"]):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            x = s["x"][a:b] if case["sorted"] else s["x"][owner[a:b]]
            y[a:b] = x.double() @ _values(s["w"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e], case["group"]).T
    return y


def _values(w, scales, zeros, group):
    n, half = w.shape
    v = torch.empty((n, 2 * half), dtype=torch.float64, device=w.device)
    v[:, 0::2] = (w % 16).double()
    v[:, 1::2] = torch.div(w, 16, rounding_mode="floor").double()
    v = v.reshape(n, -1, group)
    v = v - (8 if zeros is None else zeros.T.double().unsqueeze(2))
    return (v * scales.T.double().unsqueeze(2)).reshape(n, 2 * half)
