"""What is measured of the 8-bit integer operators: quantisation of rows, the product with scales for each token and
channel, the router of a mixture of experts and the products grouped by expert.

``own`` false computes each operator in its plain form, from elementary torch operations in float32;
``own`` true calls the framework. Both take what ``prepare`` makes.

Cases are dicts with an ``op``:
  * ``quantize`` -- rows to 8-bit codes with one scale a row, and back to the values they stand for;
  * ``matmul``   -- y = a . w^T (+ bias), 8-bit codes on both sides; ``a_form`` "float": the call quantises the activations
    itself, "codes": the caller holds them quantised; ``act`` "swiglu": of channel pairs (gate, linear);
  * ``route``    -- router scores to each token's k experts, their weights, and the assignments in expert order;
  * ``experts``  -- one product of a mixture of experts over rows grouped by expert: ``form`` "up" reads each token's row
    once for each of its experts (and applies swiglu), "down" takes rows in expert order and returns the weighted sum
    of each token's rows.
"""
import math

import torch

own = False

_T = {"float16": torch.float16, "float32": torch.float32}


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # The activations of one decoded token before a 4096-wide projection: latency.
        {"name": "quantize token", "op": "quantize", "rows": 1, "K": 4096, "dtype": "float16"},
        # A 2048-token prompt before the down projection of an 8-billion-parameter layer.
        {"name": "quantize prompt", "op": "quantize", "rows": 2048, "K": 14336, "dtype": "float16"},
        # The output projection of one decoded token: latency, and the stream of the weights.
        {"name": "matmul token", "op": "matmul", "M": 1, "N": 4096, "K": 4096, "dtype": "float16", "bias": False, "a_form": "float", "act": "none"},
        # A batch of 16 decoded tokens through the down projection.
        {"name": "matmul batch", "op": "matmul", "M": 16, "N": 4096, "K": 14336, "dtype": "float16", "bias": False, "a_form": "float", "act": "none"},
        # A prompt of 2048 tokens through the gate or up projection: the tensor cores' case.
        {"name": "matmul prompt", "op": "matmul", "M": 2048, "N": 14336, "K": 4096, "dtype": "float16", "bias": False, "a_form": "codes", "act": "none"},
        # Odd sizes in every axis, float32 activations and result, with a bias.
        {"name": "matmul odd", "op": "matmul", "M": 333, "N": 1003, "K": 4100, "dtype": "float32", "bias": True, "a_form": "float", "act": "none"},
        # One step of 64 decoded sequences before a layer of 128 experts: latency.
        {"name": "route batch", "op": "route", "T": 64, "E": 128, "k": 8, "dtype": "float16", "normalize": True},
        # Prompts of 8192 tokens in all before 256 experts; the weights keep the share of what was not chosen.
        {"name": "route prompt", "op": "route", "T": 8192, "E": 256, "k": 8, "dtype": "float32", "normalize": False},
        # One decoded token through the gate and up projections of its 8 experts of 64: the stream of their weights.
        {"name": "experts token", "op": "experts", "form": "up", "T": 1, "E": 64, "k": 8, "N": 4096, "K": 4096, "dtype": "float16", "bias": False, "skew": 0.5},
        # 64 decoded tokens through the down projection: every expert is read, for a few rows each.
        {"name": "experts batch", "op": "experts", "form": "down", "T": 64, "E": 64, "k": 8, "N": 4096, "K": 2048, "dtype": "float16", "bias": False, "skew": 0.5},
        # Prompts of 4096 tokens in all through the gate and up projections of 4 experts of 32: the tensor cores' case.
        {"name": "experts prompt", "op": "experts", "form": "up", "T": 4096, "E": 32, "k": 4, "N": 4096, "K": 4096, "dtype": "float16", "bias": False, "skew": 0.5},
        # Odd sizes in every axis, float32, biases, a few experts that most tokens want.
        {"name": "experts odd", "op": "experts", "form": "down", "T": 777, "E": 12, "k": 3, "N": 1003, "K": 1000, "dtype": "float32", "bias": True, "skew": 1.5},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "matmul", "matmul", "route", "experts", "experts", "experts"))
    dtype = rng.choice(("float16", "float16", "float32"))
    if op == "quantize":
        K = _log(rng, 64, 28672)
        return {"op": op, "rows": _log(rng, 1, min(8192, max(1, 2048 * 14336 // K))), "K": K, "dtype": dtype}
    if op == "matmul":
        while True:
            c = {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 64, 28672), "K": _log(rng, 64, 28672), "dtype": dtype,
                 "bias": rng.random() < 0.5, "a_form": rng.choice(("float", "codes")), "act": rng.choice(("none", "none", "swiglu"))}
            if c["act"] == "swiglu":
                c["N"] += c["N"] % 2
            if c["M"] * c["N"] * c["K"] <= 2048 * 14336 * 4096 and c["N"] * c["K"] <= 8192 * 28672:
                return c
    if op == "route":
        E = rng.choice((8, 16, 60, 64, 128, 160, 256, 384))
        return {"op": op, "T": _log(rng, 1, 8192 * 256 // E), "E": E, "k": rng.choice((1, 2, 4, 6, 8)), "dtype": dtype, "normalize": rng.random() < 0.6}
    while True:
        c = {"op": op, "form": rng.choice(("up", "down")), "T": _log(rng, 1, 4096), "E": rng.choice((4, 8, 12, 16, 32, 60, 64, 128)),
             "k": rng.choice((1, 2, 3, 4, 6, 8)), "N": _log(rng, 128, 8192), "K": _log(rng, 128, 8192), "dtype": dtype,
             "bias": rng.random() < 0.4, "skew": round(rng.uniform(0.0, 1.5), 2)}
        if c["form"] == "up":
            c["N"] += c["N"] % 2
        c["k"] = min(c["k"], c["E"])
        if c["T"] * c["k"] * c["N"] * c["K"] <= 16384 * 4096 * 4096 and c["E"] * c["N"] * c["K"] <= 64 * 4096 * 4096:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _activations(g, rows, K, dtype):
    """Normal values with a few channels that stand out, as a decoder's hidden states have them."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    gain = torch.where(torch.rand(K, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return (x * gain).to(dtype)


def _held(g, rows, K):
    """Codes int8 [rows, K] of normal values, each row's largest at 127, its rows 16 bytes apart at the least, and their scales."""
    held = torch.empty(rows, _ceil(K, 16) * 16, dtype=torch.int8, device="cuda")[:, :K]
    scales = torch.empty(rows, device="cuda")
    step = max(1, (64 << 20) // K)
    for i in range(0, rows, step):
        x = torch.randn(min(step, rows - i), K, generator=g, device="cuda")
        top = x.abs().amax(1, keepdim=True)
        held[i:i + step] = (x * (127.0 / top)).round_().to(torch.int8)
        scales[i:i + step] = top[:, 0] * ((torch.rand(len(x), generator=g, device="cuda") + 0.5) * K ** -0.5 / 127.0)
    return held, scales


def _scores(g, T, E, skew):
    """Router scores: normal, with experts that are wanted more than others."""
    return torch.randn(T, E, generator=g, device="cuda") + skew * torch.randn(E, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], _T[case["dtype"]]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["K"], dt)
    elif op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        s["w"], s["w_scales"] = _held(g, N, K)
        if case["a_form"] == "float":
            s["x"] = _activations(g, M, K, dt)
        else:
            s["x"], s["x_scales"] = _held(g, M, K)
            s["x_scales"] *= K ** 0.5
        s["bias"] = torch.randn(N, generator=g, device="cuda").to(dt) if case["bias"] else None
    elif op == "route":
        s["scores"] = _scores(g, case["T"], case["E"], 0.5).to(dt)
    else:
        T, E, k, N, K = (case[n] for n in ("T", "E", "k", "N", "K"))
        w, ws = _held(g, E * N, K)
        s["w"], s["w_scales"] = w.unflatten(0, (E, N)), ws.view(E, N)
        s["bias"] = torch.randn(E, N, generator=g, device="cuda").to(dt) if case["bias"] else None
        # what the router's call returns
        experts, s["weights"] = _choose(_scores(g, T, E, case["skew"]), k, True)
        s["order"], s["slots"], s["offsets"] = _group(experts, E)
        s["x"] = _activations(g, T if case["form"] == "up" else T * k, K, dt)
        if case["form"] == "down":
            s["x"] *= 0.2
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _quantize_rows(x):
    """float32 [rows, K] -> codes as float32 whole numbers, scales [rows]. Quotients in 64 bits: one in 32 can land on a border."""
    s = x.abs().amax(1) / torch.full((len(x),), 127.0, device=x.device)
    q = x.double() / s.double()[:, None]
    return torch.where(s[:, None] > 0, q, torch.zeros_like(q)).round_().clamp_(-127, 127).float(), s


def _swiglu(y):
    g, u = y[..., 0::2], y[..., 1::2]
    return g / (1 + torch.exp(-g)) * u


def _run_quantize(s):
    codes, scales = _quantize_rows(s["x"].float())
    return {"values": (codes * scales[:, None]).to(s["x"].dtype), "scales": scales}


def _codes(s):
    return _quantize_rows(s["x"].float()) if s["x"].dtype != torch.int8 else (s["x"].float(), s["x_scales"])


def _run_matmul(s):
    c = s["case"]
    a, a_scales = _codes(s)
    y = (a @ s["w"].float().t()) * a_scales[:, None] * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["act"] == "swiglu":
        y = _swiglu(y)
    return y.to(_T[c["dtype"]])


def _choose(scores, k, normalize):
    """Each token's k experts of the highest scores, ties to the lowest index, and their weights."""
    x = scores.float()
    values, at = torch.sort(x, dim=1, descending=True, stable=True)
    p = torch.exp(values - values[:, :1])
    total = (p[:, :k] if normalize else p).sum(1, keepdim=True)
    return at[:, :k].to(torch.int32), p[:, :k] / total


def _group(experts, E):
    """(order, slots, offsets): assignments (token * k + rank) in expert order, the place of each, each expert's first."""
    flat = experts.flatten().long()
    order = torch.sort(flat, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(len(flat), device=flat.device)
    counts = torch.zeros(E, dtype=torch.long, device=flat.device).index_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat((torch.zeros(1, dtype=torch.long, device=flat.device), counts.cumsum(0)))
    return order.to(torch.int32), slots.view(experts.shape).to(torch.int32), offsets.to(torch.int32)


def _run_route(s):
    c = s["case"]
    experts, weights = _choose(s["scores"], c["k"], c["normalize"])
    order, slots, offsets = _group(experts, c["E"])
    return {"experts": experts, "weights": weights, "order": order, "slots": slots, "offsets": offsets}


def _run_experts(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    rows = T * k
    a, a_scales = _quantize_rows(s["x"].float())
    off = s["offsets"].long()
    counts = off[1:] - off[:-1]
    expert = torch.repeat_interleave(torch.arange(E, device="cuda"), counts, output_size=rows)
    if c["form"] == "up":
        token = s["order"].long() // k
        a, a_scales = a[token], a_scales[token]
    # the rows of each expert that has some, padded to the most
    hit, place = torch.unique(expert, return_inverse=True)
    at = torch.arange(rows, device="cuda") - off[expert]
    padded = a.new_zeros(len(hit), int(counts.max()), c["K"])
    padded[place, at] = a
    y = torch.bmm(padded, s["w"][hit].float().transpose(1, 2))[place, at]
    y = y * a_scales[:, None] * s["w_scales"][expert]
    if s["bias"] is not None:
        y = y + s["bias"].float()[expert]
    if c["form"] == "up":
        y = _swiglu(y)
    else:
        y = (y[s["slots"].long()] * s["weights"][..., None]).sum(1)
    return y.to(_T[c["dtype"]])


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "quantize":
        return _run_quantize(state)
    if op == "matmul":
        return _run_matmul(state)
    return _run_route(state) if op == "route" else _run_experts(state)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s, op):
    from xrgpu_b200 import functional as F

    c = s["case"]
    if op == "quantize":
        codes, scales = F.int8_quantize(s["x"])
        return {"values": F.int8_dequantize(codes, scales, dtype=s["x"].dtype), "scales": scales}
    if op == "matmul":
        return F.matmul_int8(s["x"], s["w"], s["w_scales"], s["bias"], a_scales=s.get("x_scales"), activation=c["act"], dtype=_T[c["dtype"]])
    if op == "route":
        r = F.moe_route(s["scores"], c["k"], normalize=c["normalize"])
        return {"experts": r.experts, "weights": r.weights, "order": r.order, "slots": r.slots, "offsets": r.offsets}
    if c["form"] == "up":
        return F.matmul_int8_grouped(s["x"], s["w"], s["w_scales"], s["offsets"], s["bias"], order=s["order"], top_k=c["k"], activation="swiglu")
    return F.matmul_int8_grouped(s["x"], s["w"], s["w_scales"], s["offsets"], s["bias"], slots=s["slots"], weights=s["weights"])


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    es = 2 if case["dtype"] == "float16" else 4
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": 2 * n * es + 4 * case["rows"], "flops": 2 * n}
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        a = M * K * es if case["a_form"] == "float" else M * (K + 4)
        out = N // 2 if case["act"] == "swiglu" else N
        return {"bytes": a + N * (K + 4) + M * out * es + (N * es if case["bias"] else 0), "flops": 2 * M * N * K}
    T, E, k = case["T"], case["E"], case["k"]
    if op == "route":
        return {"bytes": T * E * es + T * k * 16 + 4 * (E + 1), "flops": T * E * 4}
    N, K = case["N"], case["K"]
    hit = E * (1 - (1 - k / E) ** T)  # experts that some token chose, were all wanted alike
    w = hit * N * (K + 4) + (hit * N * es if case["bias"] else 0)
    if case["form"] == "up":
        io = T * K * es + T * k * (N // 2) * es + 4 * T * k
    else:
        io = T * k * K * es + T * N * es + 8 * T * k
    return {"bytes": w + io + 4 * (E + 1), "flops": 2 * T * k * N * K}


def _exact_rows(x):
    """Values of x rounded to whole multiples of its row's scale, in float64; the scale is a float32 number of the format."""
    x = x.double()
    s = (x.abs().amax(1, keepdim=True) / 127.0).float().double()
    q = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))).clamp(-127, 127)
    return q * s, s


def _exact_experts(s):
    c = s["case"]
    T, k, N = c["T"], c["k"], c["N"]
    x = _exact_rows(s["x"])[0]
    off = s["offsets"].tolist()
    out = torch.zeros(T * k, N // 2 if c["form"] == "up" else N, dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        rows = x[(s["order"][lo:hi] // k).long()] if c["form"] == "up" else x[lo:hi]
        y = rows @ (s["w"][e].double() * s["w_scales"][e].double()[:, None]).t()
        if s["bias"] is not None:
            y += s["bias"][e].double()
        if c["form"] == "up":
            gate, linear = y[:, 0::2], y[:, 1::2]
            y = gate * torch.sigmoid(gate) * linear
        out[lo:hi] = y
    if c["form"] == "up":
        return out
    back = torch.empty(T * k, dtype=torch.long, device="cuda")
    back[s["order"].long()] = torch.arange(T * k, device="cuda")
    return torch.einsum("tkn,tk->tn", out[back].view(T, k, N), s["weights"].double())


def _exact_route(s):
    c = s["case"]
    x = s["scores"].double().cpu()
    T, E = x.shape
    k = c["k"]
    key = x.numpy()
    experts, weights = [], []
    for t in range(T):
        chosen = sorted(range(E), key=lambda e: (-key[t, e], e))[:k]
        experts.append(chosen)
        weights.append(torch.softmax(x[t, chosen] if c["normalize"] else x[t], 0)[list(range(k)) if c["normalize"] else chosen])
    flat = [e for row in experts for e in row]
    order = sorted(range(T * k), key=lambda i: (flat[i], i))
    slots = [0] * (T * k)
    for p, i in enumerate(order):
        slots[i] = p
    offsets = [0] * (E + 1)
    for e in flat:
        offsets[e + 1] += 1
    for e in range(E):
        offsets[e + 1] += offsets[e]
    whole = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"experts": whole(experts), "weights": torch.stack(weights), "order": whole(order), "slots": whole(slots).view(T, k), "offsets": whole(offsets)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        values, scales = _exact_rows(s["x"])
        return {"values": values, "scales": scales[:, 0]}
    if op == "route":
        return _exact_route(s)
    if op == "experts":
        return _exact_experts(s)
    a = _exact_rows(s["x"])[0] if case["a_form"] == "float" else s["x"].double() * s["x_scales"].double()[:, None]
    y = a @ (s["w"].double() * s["w_scales"].double()[:, None]).t()
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "swiglu":
        y = y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
    return y
