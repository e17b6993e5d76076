"""Products in 8-bit integers and the routing of tokens to experts, as measurable cases.

A case is one of four operators:

  quantise  rows of floats -> 8-bit integers with one scale for each row (``Context.quantise_i8``)
  gemm      the product of such rows with 8-bit weights, a scale for each token and channel, PReLU (``Context.gemm_i8``)
  route     logits -> the experts of every token, their weights, and the pairs in the experts' order (``Context.route``)
  experts   the product over the pairs of every expert (``Context.gemm_i8_experts``): "up" gathers the tokens' rows,
            "down" takes rows in the experts' order and sums the results of each token (``Context.combine``)

The plain forms below are elementary torch operations in 32 bits; in 64 where a rounding decides (quotients next to
a half, scores next to each other).
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_CONTEXT = None


def _framework():
    import fastertnn_b200 as ft
    global _CONTEXT
    if _CONTEXT is None:
        _CONTEXT = ft.Context(0)
    return ft, _CONTEXT


def _quantise(name, M, K, dtype):
    case = {"op": "quantise", "M": M, "K": K, "dtype": dtype}
    return dict(case, name=name) if name else case


def _gemm(name, M, K, N, dtype, alpha=1.0):
    case = {"op": "gemm", "M": M, "K": K, "N": N, "dtype": dtype, "alpha": alpha}
    return dict(case, name=name) if name else case


def _route(name, T, E, k, score, dtype, bias, groups=1, top_groups=1, group_top=1, renormalise=True, scale=1.0, pad=0.0):
    case = {"op": "route", "T": T, "E": E, "k": k, "score": score, "dtype": dtype, "bias": bias, "groups": groups,
            "top_groups": top_groups, "group_top": group_top, "renormalise": renormalise, "scale": scale, "pad": pad}
    return dict(case, name=name) if name else case


def _experts(name, form, T, E, k, K, N, dtype, alpha, skew, pad=0.0):
    case = {"op": "experts", "form": form, "T": T, "E": E, "k": k, "K": K, "N": N, "dtype": dtype, "alpha": alpha, "skew": skew, "pad": pad}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token in front of a product: the smallest call, all latency.
        _quantise("quantise_token", 1, 4096, "bf16"),
        # A prompt or a batch of features, in the library's own activation type.
        _quantise("quantise_prompt", 8192, 4096, "f32"),
        # One token through a square layer: the weights are read once, nothing else counts.
        _gemm("gemm_token", 1, 4096, 4096, "bf16"),
        # A classifier over a small batch, no size a multiple of anything.
        _gemm("gemm_classifier", 37, 1234, 1000, "f32"),
        # The fully connected layer of this library's benchmark (M = 1024, K = 4096, N = 1024) with its PReLU.
        _gemm("gemm_fc_1024", 1024, 4096, 1024, "f16", 0.5),
        # A prompt through a wide layer: the tensor pipe's case.
        _gemm("gemm_prompt", 8192, 4096, 8192, "bf16"),
        # A few sequences, one token each, softmax over a moderate number of experts.
        _route("route_step", 8, 64, 8, "softmax", "f32", False),
        # A padded batch of prompts: sigmoid scores, a bias for balance, groups, as nets with many experts have them.
        _route("route_prompt", 8191, 256, 8, "sigmoid", "bf16", True, 8, 4, 2, True, 2.5, 0.06),
        # The first product of the experts for a few tokens: some rows for some of the experts.
        _experts("experts_up_step", "up", 8, 64, 8, 2048, 1024, "bf16", 0.5, 0.0),
        # The second product of the same step, back to the tokens.
        _experts("experts_down_step", "down", 8, 64, 8, 1024, 2048, "bf16", 1.0, 0.0),
        # A padded batch of prompts with popular and unpopular experts.
        _experts("experts_up_prompt", "up", 8191, 64, 8, 2048, 1024, "bf16", 0.5, 0.7, 0.06),
        _experts("experts_down_prompt", "down", 8191, 64, 8, 1024, 2048, "bf16", 1.0, 0.7, 0.06),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        m["bytes"], m["flops"] = max(m["bytes"], w["bytes"]), max(m["flops"], w["flops"])
    while True:
        op = rng.choice(["quantise", "gemm", "gemm", "route", "experts", "experts"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        if op == "quantise":
            case = _quantise(None, _log(rng, 1, 20000), _log(rng, 64, 16384), dtype)
        elif op == "gemm":
            case = _gemm(None, _log(rng, 1, 16384), _log(rng, 64, 16384), _log(rng, 16, 16384), dtype, rng.choice([1.0, 0.5, 0.25]))
        elif op == "route":
            groups = rng.choice([1, 1, 4, 8])
            E = groups * _log(rng, 4, 384 // groups)
            top_groups = rng.randint((groups + 1) // 2, groups)
            case = _route(None, _log(rng, 1, 16384), E, rng.randint(1, min(16, top_groups * (E // groups))), rng.choice(["softmax", "sigmoid"]), dtype,
                          rng.random() < 0.5, groups, top_groups, rng.randint(1, 2), rng.random() < 0.7, rng.choice([1.0, 2.5]),
                          rng.choice([0.0, 0.1]))
        else:
            E = _log(rng, 4, 160)
            case = _experts(None, rng.choice(["up", "down"]), _log(rng, 1, 8192), E, rng.randint(1, min(8, E)), _log(rng, 64, 4096), _log(rng, 64, 4096),
                            dtype, rng.choice([1.0, 0.5]), rng.choice([0.0, 0.7]), rng.choice([0.0, 0.1]))
            if E * case["K"] * case["N"] > 300e6:
                continue
        w = work(case)
        if w["bytes"] <= most[op]["bytes"] and w["flops"] <= most[op]["flops"]:
            return case


def _pitch(K):
    """Bytes from one row of 8-bit integers to the next."""
    return (K + 15) // 16 * 16


def _floats(g, M, K, dtype):
    """Activations: a few channels far larger than the rest, an empty row now and then."""
    x = torch.randn(M, K, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(K, generator=g, device="cuda")) * (1 + 9 * (torch.rand(K, generator=g, device="cuda") < 0.01))
    if M > 16:
        x[torch.rand(M, generator=g, device="cuda") < 0.01] = 0
    return x.to(_DT[dtype])


def _int8(g, *shape):
    return (32 * torch.randn(*shape, generator=g, device="cuda")).round_().clamp_(-127, 127).to(torch.int8)


def _rows8(g, M, K):
    """Quantised rows with room behind each row up to a multiple of 16 bytes, and their scales."""
    q = torch.zeros(M, _pitch(K), dtype=torch.int8, device="cuda")
    q[:, :K] = _int8(g, M, K)
    return q, torch.rand(M, generator=g, device="cuda") * 0.05 + 0.01


def _scales(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda") * 2e-3 + 1e-4


def _plan(experts, E):
    """The pairs (token, j) in the experts' order: offsets of the experts, the token of every place, the place of every pair."""
    T, k = experts.shape
    flat = experts.reshape(-1)
    key, order = torch.sort(torch.where(flat < 0, E, flat), stable=True)
    place = torch.arange(T * k, device=flat.device)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=flat.device, dtype=key.dtype))
    rows = torch.where(key < E, order // k, -1)
    slots = torch.empty(T * k, dtype=torch.int64, device=flat.device)
    slots[order] = torch.where(key < E, place, -1)
    return offsets.to(torch.int32), rows.to(torch.int32), slots.reshape(T, k).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "quantise":
        s["x"] = _floats(g, case["M"], case["K"], case["dtype"])
        s["q"] = torch.empty(case["M"], _pitch(case["K"]), dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["M"], dtype=torch.float32, device="cuda")
    elif op == "gemm":
        s["q"], s["scale"] = _rows8(g, case["M"], case["K"])
        s["w"], s["w_scale"] = _int8(g, case["N"], case["K"]), _scales(g, case["N"])
        s["y"] = torch.empty(case["M"], case["N"], dtype=_DT[case["dtype"]], device="cuda")
        if own:
            s["handle"] = _framework()[1].upload_weights_i8(s["w"].data_ptr(), s["w_scale"].data_ptr(), case["N"], case["K"])
    elif op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        x = torch.randn(T, E, generator=g, device="cuda") * 1.5 + 0.5 * torch.randn(E, generator=g, device="cuda")
        x[T - int(T * case["pad"]):] = -math.inf  # the tokens behind the last sequence go to no expert
        s["logits"] = x.to(_DT[case["dtype"]])
        s["bias"] = torch.randn(E, generator=g, device="cuda") * 0.1 if case["bias"] else None
        for key, shape, dt in (("experts", (T, k), torch.int32), ("weights", (T, k), torch.float32), ("offsets", (E + 1,), torch.int32),
                               ("rows", (T * k,), torch.int32), ("slots", (T, k), torch.int32)):
            s[key] = torch.empty(shape, dtype=dt, device="cuda")
        if own:
            ft, _ = _framework()
            s["route"] = ft.Route(experts=E, top_k=k, score=ft.ROUTE_SIGMOID if case["score"] == "sigmoid" else ft.ROUTE_SOFTMAX, groups=case["groups"],
                                  top_groups=case["top_groups"], group_top=case["group_top"], renormalise=int(case["renormalise"]), scale=case["scale"])
    else:
        T, E, k, K, N = (case[n] for n in "TEkKN")
        liking = torch.randn(T, E, generator=g, device="cuda") + case["skew"] * torch.randn(E, generator=g, device="cuda")
        experts = torch.topk(liking, k, dim=1).indices
        experts[T - int(T * case["pad"]):] = -1
        s["offsets"], s["rows"], s["slots"] = _plan(experts, E)
        s["bounds"] = s["offsets"].tolist()
        s["weights"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), 1)
        s["q"], s["scale"] = _rows8(g, T if case["form"] == "up" else T * k, K)
        s["w"], s["w_scale"] = _int8(g, E, N, K), _scales(g, E, N)
        s["y"] = torch.zeros(T * k, N, dtype=_DT[case["dtype"]], device="cuda")
        s["out"] = torch.empty(T, N, dtype=_DT[case["dtype"]], device="cuda")
        if own:
            s["handle"] = _framework()[1].upload_weights_i8(s["w"].data_ptr(), s["w_scale"].data_ptr(), N, K, experts=E)
            if case["form"] == "down":  # products that are still to be summed keep 32 bits: the sum is what is rounded
                s["y"] = s["y"].float()
    return s


# --------------------------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------------------------

def _run_own(s):
    ft, ctx = _framework()
    case, op = s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    dt = {"f32": ft.F32, "f16": ft.F16, "bf16": ft.BF16}[case["dtype"]]
    if op == "quantise":
        ctx.quantise_i8(s["x"].data_ptr(), dt, s["q"].data_ptr(), s["scale"].data_ptr(), case["M"], case["K"], stream=stream)
        return s["q"][:, :case["K"]], s["scale"]
    if op == "gemm":
        ctx.gemm_i8(s["handle"], s["q"].data_ptr(), s["scale"].data_ptr(), s["y"].data_ptr(), dt, case["M"], case["alpha"], stream=stream)
        return s["y"]
    if op == "route":
        ctx.route(s["route"], s["logits"].data_ptr(), dt, 0 if s["bias"] is None else s["bias"].data_ptr(), case["T"], s["experts"].data_ptr(),
                  s["weights"].data_ptr(), s["offsets"].data_ptr(), s["rows"].data_ptr(), s["slots"].data_ptr(), stream=stream)
        return s["experts"], s["weights"], s["offsets"], s["rows"], s["slots"]
    up = case["form"] == "up"
    ctx.gemm_i8_experts(s["handle"], s["q"].data_ptr(), s["scale"].data_ptr(), s["rows"].data_ptr() if up else 0, s["offsets"].data_ptr(),
                        s["y"].data_ptr(), dt if up else ft.F32, s["q"].shape[0], case["T"] * case["k"], case["alpha"], stream=stream)
    if up:
        return s["y"]
    ctx.combine(s["y"].data_ptr(), ft.F32, case["T"] * case["k"], s["slots"].data_ptr(), s["weights"].data_ptr(), case["k"], s["out"].data_ptr(), dt,
                case["T"], case["N"], stream=stream)
    return s["out"]


# --------------------------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------------------------

def _prelu(y, alpha):
    return torch.where(y > 0, y, y * alpha)


def _plain_quantise(x):
    x = x.double()  # which integer is nearest has to be decided on the true quotient
    most = x.abs().amax(1, keepdim=True)
    q = torch.where(most > 0, torch.round(x * 127 / most), 0.0)
    return q.to(torch.int8), (most / 127).float().squeeze(1)


def _plain_route(case, logits, bias):
    E, k, G = case["E"], case["k"], case["groups"]
    x = logits.double()  # scores that lie next to each other have to come out in their true order
    off = torch.isneginf(x)
    if case["score"] == "sigmoid":
        p = torch.where(off, 0.0, 1 / (1 + torch.exp(-x)))
    else:
        top = x.amax(1, keepdim=True)
        p = torch.where(off, 0.0, torch.exp(x - torch.where(torch.isinf(top), 0.0, top)))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
    biased = p if bias is None else p + bias.double()
    key = torch.where(off, -math.inf, x if bias is None else biased)
    if case["top_groups"] < G:
        if case["group_top"] == 1:
            worth = key.reshape(-1, G, E // G).amax(2)
        else:
            two = torch.sort(torch.where(off, -math.inf, biased).reshape(-1, G, E // G), dim=2, descending=True).values[:, :, :2]
            worth = torch.where(torch.isinf(two[:, :, 0]), -math.inf, torch.where(torch.isinf(two), 0.0, two).sum(2))
        best = torch.sort(worth, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(worth).scatter(1, best, 1.0) > 0
        key = torch.where(kept.repeat_interleave(E // G, 1), key, -math.inf)
    value, chosen = torch.sort(key, dim=1, descending=True, stable=True)
    value, chosen = value[:, :k], chosen[:, :k]
    w = torch.where(torch.isinf(value), 0.0, p.gather(1, chosen))
    if case["renormalise"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    experts = torch.where(torch.isinf(value), -1, chosen)
    return (experts.to(torch.int32), (w * case["scale"]).float(), *_plan(experts, E))


def run(state):
    if own:
        return _run_own(state)
    s, case, op = state, state["case"], state["case"]["op"]
    if op == "quantise":
        return _plain_quantise(s["x"])
    if op == "route":
        return _plain_route(case, s["logits"], s["bias"])
    K, dt = case["K"], _DT[case["dtype"]]
    if op == "gemm":
        y = s["q"][:, :K].float() @ s["w"].float().T
        return _prelu(y * s["scale"][:, None] * s["w_scale"], case["alpha"]).to(dt)
    T, k, N = case["T"], case["k"], case["N"]
    y = torch.zeros(T * k, N, device="cuda")
    for e, (a, b) in enumerate(zip(s["bounds"], s["bounds"][1:])):
        if a == b:
            continue
        r = s["rows"][a:b].long() if case["form"] == "up" else slice(a, b)
        y[a:b] = _prelu((s["q"][r, :K].float() @ s["w"][e].float().T) * s["scale"][r][:, None] * s["w_scale"][e], case["alpha"])
    if case["form"] == "up":
        return y.to(dt)
    at = s["slots"].long()
    return (torch.where(at < 0, 0.0, s["weights"])[:, :, None] * y[at.clamp(min=0)]).sum(1).to(dt)


# --------------------------------------------------------------------------------------------
# what one pass cannot do without, and the definitions in 64 bits
# --------------------------------------------------------------------------------------------

def work(case):
    op, b = case["op"], _BYTES[case["dtype"]]
    if op == "quantise":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (b + 1) + 4 * M, "flops": 3 * M * K}
    if op == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * b, "flops": 2 * M * N * K}
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * b + (4 * E if case["bias"] else 0) + 16 * T * k + 4 * (E + 1), "flops": 4 * T * E}
    T, E, k, K, N = (case[n] for n in "TEkKN")
    T -= int(T * case["pad"])
    met = E * (1 - (1 - k / E) ** T)  # experts that get a row, for choices that are all alike
    rows = T if case["form"] == "up" else T * k
    wrote = T * k if case["form"] == "up" else T
    return {"bytes": int(rows * (K + 4) + met * N * (K + 4) + wrote * N * b + 8 * T * k), "flops": 2 * T * k * N * K}


def _exact_product(q, scale, w, w_scale, alpha):
    y = (q.double() @ w.double().T) * scale.double().unsqueeze(1) * w_scale.double().unsqueeze(0)
    return torch.maximum(y, torch.zeros_like(y)) + alpha * torch.minimum(y, torch.zeros_like(y))


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantise":
        x = s["x"].double().cpu().numpy()
        a = np.max(np.abs(x), axis=1)
        q = np.rint(np.divide(x * 127.0, a[:, None], out=np.zeros_like(x), where=a[:, None] > 0))
        return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(a / 127.0)
    if op == "gemm":
        return _exact_product(s["q"][:, :case["K"]], s["scale"], s["w"], s["w_scale"], case["alpha"])
    if op == "experts":
        T, k, K, N, up = case["T"], case["k"], case["K"], case["N"], case["form"] == "up"
        rows, q, b = s["rows"].cpu().numpy(), s["q"][:, :K], s["bounds"]
        result = torch.zeros(T * k if up else T, N, dtype=torch.float64, device="cuda")
        place = torch.full((T * k,), -1, dtype=torch.int64)
        flat = s["slots"].reshape(-1).cpu().long()
        pairs = torch.nonzero(flat >= 0).squeeze(1)
        place[flat[pairs]] = pairs
        for e in range(case["E"]):
            if b[e + 1] > b[e]:
                at = torch.from_numpy(rows[b[e]:b[e + 1]].astype(np.int64)) if up else torch.arange(b[e], b[e + 1])
                at = at.cuda()
                y = _exact_product(q[at], s["scale"][at], s["w"][e], s["w_scale"][e], case["alpha"])
                if up:
                    result[b[e]:b[e + 1]] = y
                else:
                    pair = place[b[e]:b[e + 1]].cuda()
                    result.index_add_(0, pair // k, y * s["weights"].reshape(-1)[pair].double()[:, None])
        return result
    # route: one token after the other
    x = s["logits"].double().cpu().numpy()
    bias = None if s["bias"] is None else s["bias"].double().cpu().numpy()
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    size = E // G
    experts, weights = np.full((T, k), -1, np.int32), np.zeros((T, k))
    by_expert = [[] for _ in range(E)]
    for t in range(T):
        there = np.flatnonzero(x[t] != -np.inf)
        if not there.size:
            continue
        p = np.zeros(E)
        v = x[t, there]
        if case["score"] == "sigmoid":
            p[there] = 1.0 / (1.0 + np.exp(-v))
        else:
            e = np.exp(v - v.max())
            p[there] = e / e.sum()
        worth = p if bias is None else p + bias
        rank = x[t] if bias is None else worth
        if case["top_groups"] < G:
            of_group = []
            for i in range(G):
                inside = there[there // size == i]
                if inside.size:
                    of_group.append((-(rank[inside].max() if case["group_top"] == 1 else np.sort(worth[inside])[-2:].sum()), i))
            kept = {i for _, i in sorted(of_group)[:case["top_groups"]]}
            there = np.array([i for i in there if i // size in kept])
        chosen = there[np.lexsort((there, -rank[there]))][:k]
        total = p[chosen].sum() + 1e-20 if case["renormalise"] else 1.0
        experts[t, :len(chosen)] = chosen
        weights[t, :len(chosen)] = case["scale"] * p[chosen] / total
        for j, i in enumerate(chosen):
            by_expert[i].append((t, j))
    offsets, rows, slots, at = [0], np.full(T * k, -1, np.int32), np.full((T, k), -1, np.int32), 0
    for pairs in by_expert:
        for t, j in pairs:
            rows[at], slots[t, j] = t, at
            at += 1
        offsets.append(at)
    return (torch.from_numpy(experts), torch.from_numpy(weights), torch.tensor(offsets, dtype=torch.int32), torch.from_numpy(rows), torch.from_numpy(slots))
