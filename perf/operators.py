"""What is measured of the block-scaled serving operators: microscaled 4-bit floating point (quantisation and
product) and the attention over a key/value cache held in 8 bits (with the append that fills it).

``own`` false computes each operator in its plain form, from elementary torch operations in float32;
``own`` true calls the framework. Both take what ``prepare`` makes.

Cases are dicts with an ``op``:
  * ``quantize``  -- activations to 4-bit codes with one power-of-two scale per 32, and back to the values they stand for;
  * ``matmul``    -- y = a . w^T (+ bias) with both operands in that form; ``a_form`` "float": the call quantises the
    activations itself, "codes": the caller holds them quantised;
  * ``append``    -- new keys and values into the paged 8-bit cache, then the values that the touched pages hold;
  * ``attention`` -- queries over the paged 8-bit cache, one token per sequence or prompts.
"""
import math
import random

import torch

own = False

_T = {"float16": torch.float16, "float32": torch.float32}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_LIMIT = {"int8": 127.0, "e4m3": 448.0}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # The activations of one decoded token before a 4096-wide projection: latency.
        {"name": "quantize token", "op": "quantize", "rows": 1, "K": 4096, "dtype": "float16"},
        # A 2048-token prompt before the down projection of an 8-billion-parameter layer.
        {"name": "quantize prompt", "op": "quantize", "rows": 2048, "K": 14336, "dtype": "float16"},
        # The output projection of one decoded token: latency, and the stream of 4-bit weights.
        {"name": "matmul token", "op": "matmul", "M": 1, "N": 4096, "K": 4096, "dtype": "float16", "bias": False, "a_form": "float"},
        # A batch of 16 decoded tokens through the gate or up projection.
        {"name": "matmul batch", "op": "matmul", "M": 16, "N": 14336, "K": 4096, "dtype": "float16", "bias": False, "a_form": "float"},
        # A prompt of 2048 tokens through the same projection: the tensor cores' case.
        {"name": "matmul prompt", "op": "matmul", "M": 2048, "N": 14336, "K": 4096, "dtype": "float16", "bias": False, "a_form": "codes"},
        # Odd sizes in every axis, float32 activations and result, with a bias.
        {"name": "matmul odd", "op": "matmul", "M": 333, "N": 1003, "K": 4100, "dtype": "float32", "bias": True, "a_form": "float"},
        # One decoded token of each of 64 sequences into the cache.
        {"name": "append tokens", "op": "append", "B": 64, "new": 1, "past": 2000, "ragged": True, "Hkv": 8, "D": 128,
         "page": 64, "code": "int8", "dtype": "float16"},
        # Five ragged prompts (chunks of a chunked prefill) into the cache.
        {"name": "append prompts", "op": "append", "B": 5, "new": 1700, "past": 1000, "ragged": True, "Hkv": 8, "D": 128,
         "page": 32, "code": "e4m3", "dtype": "float16"},
        # One decoded token of one sequence: latency.
        {"name": "attend token", "op": "attention", "B": 1, "new": 1, "past": 2047, "ragged": False, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "code": "int8", "dtype": "float16", "window": 0},
        # A batch of long sequences, ragged: the stream of the cache. 64 query heads on 8 key/value heads.
        {"name": "attend batch", "op": "attention", "B": 32, "new": 1, "past": 16000, "ragged": True, "Hq": 64, "Hkv": 8,
         "D": 128, "page": 64, "code": "int8", "dtype": "float16", "window": 0},
        # Two ragged chunks of prompts on top of what the cache holds: the tensor cores' case.
        {"name": "attend prompts", "op": "attention", "B": 2, "new": 4096, "past": 4096, "ragged": True, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "code": "int8", "dtype": "float16", "window": 0},
        # A few tokens a sequence (speculative decoding), float32, small heads and pages, odd groups, a sliding window.
        {"name": "attend odd", "op": "attention", "B": 7, "new": 5, "past": 900, "ragged": True, "Hq": 15, "Hkv": 3,
         "D": 64, "page": 16, "code": "e4m3", "dtype": "float32", "window": 333},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "matmul", "matmul", "append", "attention", "attention"))
    dtype = rng.choice(("float16", "float16", "float32"))
    if op == "quantize":
        K = _log(rng, 64, 28672)
        return {"op": op, "rows": _log(rng, 1, min(8192, max(1, 2048 * 14336 // K))), "K": K, "dtype": dtype}
    if op == "matmul":
        while True:
            c = {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 64, 28672), "K": _log(rng, 64, 28672), "dtype": dtype,
                 "bias": rng.random() < 0.5, "a_form": rng.choice(("float", "codes"))}
            if c["M"] * c["N"] * c["K"] <= 2048 * 14336 * 4096 and c["N"] * c["K"] <= 8192 * 28672:
                return c
    c = {"op": op, "ragged": rng.random() < 0.7, "Hkv": rng.choice((1, 2, 4, 8)), "D": rng.choice((64, 128)),
         "page": rng.choice((16, 32, 64, 128)), "code": rng.choice(("int8", "e4m3")), "dtype": dtype}
    if op == "append":
        c.update(B=_log(rng, 1, 64))
        c.update(new=_log(rng, 1, max(1, 8000 // c["B"])), past=_log(rng, 1, 4000))
        return c
    c["Hq"] = c["Hkv"] * rng.choice((1, 2, 3, 4, 8))
    c["window"] = rng.choice((0, 0, 0, _log(rng, 16, 4096)))
    if rng.random() < 0.5:  # one token, or the few of speculative decoding
        c.update(B=_log(rng, 1, 64), new=rng.choice((1, 1, 1, 2, 5)))
        c["past"] = _log(rng, 1, max(1, 32 * 16000 // c["B"] // 2)) if c["B"] > 8 else _log(rng, 1, 32000)
    else:
        c.update(B=rng.choice((1, 2, 3)) if c["Hq"] <= 32 else 1, new=_log(rng, 6, 1500))
        c["past"] = _log(rng, 1, 2500)
    return c


def _lengths(case):
    """(new, total) tokens of each sequence, from the case alone so that work() knows them too."""
    rng = random.Random(case["B"] * 1000003 + case["new"] * 10007 + case["past"])
    new, total = [], []
    for _ in range(case["B"]):
        n, p = case["new"], case["past"]
        if case["ragged"]:
            n = max(1, int(n * rng.uniform(0.4, 1.0) + 0.5))
            p = int(p * rng.uniform(0.1, 1.0))
        new.append(n)
        total.append(n + p)
    return new, total


# ------------------------------------------------------------------------------------------------ inputs
def _activations(g, rows, K, dtype):
    """Normal values with a few channels that stand out, as a decoder's hidden states have them."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    gain = torch.where(torch.rand(K, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return (x * gain).to(dtype)


def _tile(scales):
    """[rows, kb] scale bytes in tiles of 128 rows and 4 blocks: [rows/128, kb/4, 32, 4, 4], padded with zeros."""
    rows, kb = scales.shape
    R, C = _ceil(rows, 128), _ceil(kb, 4)
    p = torch.zeros(R * 128, C * 4, dtype=torch.uint8, device=scales.device)
    p[:rows, :kb] = scales
    return p.view(R, 4, 32, C, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile(tiled, rows, kb):
    R, C = tiled.shape[:2]
    return tiled.permute(0, 3, 2, 1, 4).reshape(R * 128, C * 4)[:rows, :kb]


def _pages(case, g):
    """A cache in use: pages in no order, what a page's scale and codes are after real appends, and left-over
    codes of earlier sequences behind each sequence's last token."""
    new, total = _lengths(case)
    page, Hkv, D, B = case["page"], case["Hkv"], case["D"], case["B"]
    need = [_ceil(t, page) for t in total]
    P = sum(need) + 3
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    host = order.cpu()
    for b, n in enumerate(need):
        table[b, :n] = host[at:at + n]
        at += n

    def side():
        scale = (torch.rand(P, Hkv, generator=g, device="cuda") * 1.5 + 0.5) * 3.5 / _LIMIT[case["code"]]
        codes = torch.empty(P, Hkv, page, D, dtype=_CODE[case["code"]], device="cuda")
        step = max(1, (64 << 20) // (Hkv * page * D))
        for i in range(0, P, step):
            x = torch.randn(min(step, P - i), Hkv, page, D, generator=g, device="cuda") * (_LIMIT[case["code"]] / 3.5)
            x = x.clamp_(-_LIMIT[case["code"]], _LIMIT[case["code"]])
            codes[i:i + step] = x.round_().to(torch.int8) if case["code"] == "int8" else x.to(torch.float8_e4m3fn)
        return codes, scale

    k, ks = side()
    v, vs = side()
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
    return {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs, "page_table": table.cuda(), "cu_seqlens": cu.cuda(),
            "kv_len": torch.tensor(total, dtype=torch.int32).cuda(), "T": sum(new)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], _T[case["dtype"]]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["K"], dt)
    elif op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        w = torch.randn(N, K, generator=g, device="cuda") * (K ** -0.5)
        s["w"], ws = _quantize_rows(w)
        s["w_scales"] = _tile(ws)
        del w
        x = _activations(g, M, K, dt)
        if case["a_form"] == "float":
            s["x"] = x
        else:
            s["x"], xs = _quantize_rows(x.float())
            s["x_scales"] = _tile(xs)
        s["bias"] = torch.randn(N, generator=g, device="cuda").to(dt) if case["bias"] else None
    else:
        s.update(_pages(case, g))
        T = s["T"]
        if op == "append":
            s["k"] = (torch.randn(T, case["Hkv"], case["D"], generator=g, device="cuda") * 1.2).to(dt)
            s["v"] = (torch.randn(T, case["Hkv"], case["D"], generator=g, device="cuda") * 1.2).to(dt)
            # the tokens of the pages that the append touches: each sequence's last ones
            new, total = _lengths(case)
            back = [total[b] - (total[b] - n) // case["page"] * case["page"] for b, n in enumerate(new)]
            s["back_cu"] = torch.tensor([0] + back, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
            s["back_T"] = sum(back)
        else:
            s["q"] = torch.randn(T, case["Hq"], case["D"], generator=g, device="cuda").to(dt)
            s["max_new"] = max(_lengths(case)[0])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _power(e):
    """2^e in float32 for whole e in [-127, 127], exactly, from its bits (2^-127 is a subnormal)."""
    return torch.where(e > -127, (e.to(torch.int32) + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantize_rows(x):
    """float32 [rows, K] -> packed codes uint8 [rows, kb, 16] and scale bytes uint8 [rows, kb]."""
    rows, K = x.shape
    kb = _ceil(K, 32)
    p = torch.nn.functional.pad(x, (0, kb * 32 - K)).view(rows, kb, 32)
    a = p.abs().amax(-1)
    bad = ~torch.isfinite(a)
    _, e = torch.frexp(torch.where(bad, 1.0, a))  # a = m 2^e, 0.5 <= m < 1: floor(log2 a) = e - 1
    E = torch.where(a > 0, e.to(torch.int32) - 3, torch.full_like(e, -127, dtype=torch.int32)).clamp(-127, 127)
    v = p * _power(-E)[..., None]
    m = v.abs()
    # round to nearest, ties to the even code: the borders that go up are those above an odd code
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8) + (m >= 1.75).to(torch.uint8)
            + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8) + (m > 5.0).to(torch.uint8))
    code = code + torch.signbit(p).to(torch.uint8) * 8
    code = torch.where(bad[..., None], 0, code).to(torch.uint8).view(rows, kb, 16, 2)
    byte = torch.where(bad, 255, E + 127).to(torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), byte


def _values(codes, scales, K):
    """Packed codes [rows, kb, 16] and scale bytes [rows, kb] -> float32 [rows, K]."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int32)
    s = torch.where(scales == 255, float("nan"), _power(scales.to(torch.int32) - 127))
    return (table[c] * s[..., None]).flatten(1)[:, :K]


def _run_quantize(s):
    c, x = s["case"], s["x"]
    codes, scales = _quantize_rows(x.float())
    return _values(codes, scales, c["K"]).to(x.dtype)


def _run_matmul(s):
    c = s["case"]
    M, N, K = c["M"], c["N"], c["K"]
    kb = _ceil(K, 32)
    if c["a_form"] == "float":
        ac, asc = _quantize_rows(s["x"].float())
    else:
        ac, asc = s["x"], _untile(s["x_scales"], M, kb)
    y = _values(ac, asc, K) @ _values(s["w"], _untile(s["w_scales"], N, kb), K).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(_T[c["dtype"]])


def _round_code(x, kind):
    """float64 values to codes: nearest, ties to even. In 64 bits, since a quotient in 32 can land on a border."""
    if kind == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    _, e = torch.frexp(x)
    step = _power64((e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448).float().to(torch.float8_e4m3fn)


def _power64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _row_index(cu, kv_len, T):
    """(sequence, position) of each of the T token rows."""
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    return b, (kv_len.long() - (cu[1:] - cu[:-1]).long())[b] + t - cu.long()[b]


def _append_side(s, x, cache, scale):
    """One side (keys or values) of the append, for all pages and tokens at once."""
    c = s["case"]
    page, P, Hkv = c["page"], cache.shape[0], c["Hkv"]
    cu, kv_len = s["cu_seqlens"], s["kv_len"]
    b, pos = _row_index(cu, kv_len, x.shape[0])
    pid = s["page_table"][b, pos // page].long()
    xf = x.float()
    new = torch.zeros(P, Hkv, device=x.device).index_reduce_(0, pid, xf.abs().amax(-1), "amax")
    new = new / torch.full_like(new, _LIMIT[c["code"]])
    # pages that hold older tokens: the first touched page of each sequence, unless it starts with a new token
    n = (cu[1:] - cu[:-1]).long()
    start = kv_len.long() - n
    first = s["page_table"][torch.arange(len(n), device=x.device), (start // page).clamp(max=s["page_table"].shape[1] - 1)].long()
    older = (start % page != 0) & (n > 0)
    touched = torch.zeros(P, dtype=torch.bool, device=x.device)
    touched[pid] = True
    held = torch.zeros(P, dtype=torch.bool, device=x.device)
    held[first[older]] = True
    old = torch.where(held[:, None], scale, torch.zeros_like(scale))
    now = torch.where(touched[:, None], torch.maximum(old, new), scale)
    grown = first[older]
    up = (now[grown] > old[grown])[..., None, None]
    was = cache[grown]
    wf = was.float().double()
    was_s, now_s = old[grown].double()[..., None, None], now[grown].double()[..., None, None]
    cache[grown] = _round_code(torch.where(up, wf * was_s / now_s, wf), c["code"])
    st = now[pid].double()[..., None]
    cache[pid, :, pos % page] = _round_code(torch.where(st > 0, xf.double() / st, torch.zeros_like(st)), c["code"])
    scale.copy_(now)


def _read_side(s, cache, scale, cu, T):
    b, pos = _row_index(cu, s["kv_len"], T)
    page = s["case"]["page"]
    pid = s["page_table"][b, pos // page].long()
    return (cache[pid, :, pos % page].float() * scale[pid][..., None]).to(_T[s["case"]["dtype"]])


def _run_append(s):
    _append_side(s, s["k"], s["k_cache"], s["k_scale"])
    _append_side(s, s["v"], s["v_cache"], s["v_scale"])
    k = _read_side(s, s["k_cache"], s["k_scale"], s["back_cu"], s["back_T"])
    v = _read_side(s, s["v_cache"], s["v_scale"], s["back_cu"], s["back_T"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gather(s, cache, scale, to):
    """The cache of all sequences, padded to the longest: [B, Hkv, tokens, D] in `to`."""
    t = s["page_table"].clamp(min=0).long()
    x = cache[t].to(to) * scale[t].to(to)[..., None, None]  # [B, pages, Hkv, page, D]
    B, n, Hkv, page, D = x.shape
    return x.transpose(1, 2).reshape(B, Hkv, n * page, D)


def _attend(s, to):
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    G, L = Hq // Hkv, s["max_new"]
    cu, kv_len = s["cu_seqlens"].long(), s["kv_len"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(L, device="cuda")
    real = i[None] < n[:, None]
    rows = (cu[:-1, None] + i[None]).clamp(max=s["T"] - 1)  # [B, L]
    q = s["q"][rows].to(to).view(B, L, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * L, D)
    x = (q @ _gather(s, s["k_cache"], s["k_scale"], to).transpose(-1, -2)).view(B, Hkv, G, L, -1) * (D ** -0.5)
    at = torch.arange(x.shape[-1], device="cuda")
    pos = (kv_len - n)[:, None] + i[None]
    seen = (at <= pos[..., None]) & (at < kv_len[:, None, None])
    if c["window"]:
        seen &= at > pos[..., None] - c["window"]
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, G * L, -1) @ _gather(s, s["v_cache"], s["v_scale"], to)).view(B, Hkv, G, L, D)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, L, Hq, D)[real]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "quantize":
        return _run_quantize(state)
    if op == "matmul":
        return _run_matmul(state)
    if op == "append":
        return _run_append(state)
    return _attend(state, torch.float32).to(_T[state["case"]["dtype"]])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s, op):
    from xrgpu_b200 import functional as F

    c = s["case"]
    if op == "quantize":
        codes, scales = F.mxfp4_quantize(s["x"])
        return F.mxfp4_dequantize(codes, scales, K=c["K"], dtype=s["x"].dtype)
    if op == "matmul":
        return F.matmul_mxfp4(s["x"], s["w"], s["w_scales"], s["bias"], a_scales=s.get("x_scales"), K=c["K"],
                              dtype=_T[c["dtype"]])
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["page_table"])
    if op == "append":
        F.kv8_append(s["k"], s["v"], *cache, s["cu_seqlens"], s["kv_len"])
        k, v = F.kv8_read(*cache, s["back_cu"], s["kv_len"], rows=s["back_T"], dtype=s["k"].dtype)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return F.attention_kv8(s["q"], *cache, s["cu_seqlens"], s["kv_len"], window=c["window"])


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    es = 2 if case["dtype"] == "float16" else 4
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": 2 * n * es, "flops": 2 * n}
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        a = M * K * es if case["a_form"] == "float" else M * K * 17 / 32
        return {"bytes": a + N * K * 17 / 32 + M * N * es + (N * es if case["bias"] else 0), "flops": 2 * M * N * K}
    new, total = _lengths(case)
    per = case["Hkv"] * case["D"]
    if op == "append":
        page = case["page"]
        back = sum(t - (t - n) // page * page for n, t in zip(new, total))
        return {"bytes": 2 * (sum(new) * per * (es + 1) + back * per * es), "flops": 4 * sum(new) * per}
    pairs, tokens = 0, 0
    for n, t in zip(new, total):
        w = case["window"] or t
        tokens += min(t, w + n - 1)
        # row i sees min(position + 1, window) tokens
        first = t - n + 1
        short = max(0, min(n, w - first))
        pairs += short * first + short * (short - 1) // 2 + (n - short) * w
    q = sum(new) * case["Hq"] * case["D"]
    pages = sum(_ceil(t, case["page"]) for t in total)
    return {"bytes": 2 * tokens * per + 2 * q * es + 8 * pages * case["Hkv"], "flops": 4 * pairs * case["Hq"] * case["D"]}


def _exact_rows(x):
    """Values of x rounded to blocks of 32 4-bit numbers, in float64: the nearest representable, ties to the even code."""
    rows, K = x.shape
    kb = _ceil(K, 32)
    p = torch.zeros(rows, kb * 32, dtype=torch.float64, device=x.device)
    p[:, :K] = x.double()
    p = p.view(rows, kb, 32)
    a = p.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(a.clamp(min=1e-300))  # floor(log2 a) = e - 1
    unit = _power64((e - 3).clamp(-127, 127))
    m = (p / unit).abs().clamp(max=6.0)
    # the spacing of the numbers at m: 0.5 below 2, 1 below 4, 2 above; torch.round takes ties to even multiples,
    # which are the even codes
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).to(torch.float64)
    q = torch.round(m / step) * step
    return (torch.sign(p) * q * unit).view(rows, kb * 32)[:, :K]


def _exact_held(codes, tiled, rows, K):
    kb = _ceil(K, 32)
    byte = _untile(tiled, rows, kb).double()
    n = codes.view(rows, kb, 16, 1) >> torch.tensor([0, 4], dtype=torch.uint8, device=codes.device)
    n = (n & 15).reshape(rows, kb, 32).double()
    mag = n % 8
    v = torch.where(mag < 4, mag / 2, torch.where(mag < 6, mag - 2, mag * 2 - 8))
    return ((1 - 2 * (n >= 8).double()) * v * _power64(byte - 127)[..., None]).view(rows, kb * 32)[:, :K]


def _exact_append(s):
    c = s["case"]
    L, page = _LIMIT[c["code"]], c["page"]
    new, total = _lengths(c)
    cu = s["cu_seqlens"].tolist()
    table = s["page_table"].tolist()
    out = {}
    for side in ("k", "v"):
        x = s[side].double()
        cache, scale = s[side + "_cache"].double() if c["code"] == "int8" else s[side + "_cache"].float().double(), s[side + "_scale"].double().clone()
        back = []
        for b in range(c["B"]):
            start = total[b] - new[b]
            for j in range(start // page, _ceil(total[b], page)):
                lo, hi = max(start, j * page), min(total[b], (j + 1) * page)
                rows = x[cu[b] + lo - start:cu[b] + hi - start].transpose(0, 1)  # [Hkv, n, D]
                pid, held = table[b][j], lo - j * page
                # the quotient is a float32 number of the cache's state: rounded like one
                a = (rows.abs().amax((1, 2)) / L).float().double()
                old = scale[pid] if held else torch.zeros_like(a)
                now = torch.maximum(old, a)
                tok = torch.cat((cache[pid, :, :held] * old[:, None, None] / now[:, None, None], rows / now[:, None, None]), 1)
                if c["code"] == "int8":
                    tok = torch.round(tok).clamp(-L, L)
                else:
                    t = tok.abs().clamp(max=L)
                    step = _power64(torch.frexp(t.clamp(min=2.0 ** -6))[1] - 4)
                    tok = torch.sign(tok) * (torch.round(t / step) * step).clamp(max=L)
                scale[pid] = now
                back.append((tok * now[:, None, None]).transpose(0, 1))
        out[side], out[side + "_scale"] = torch.cat(back), scale
    return {n: out[n] for n in ("k", "v", "k_scale", "v_scale")}


def _exact_attention(s):
    c = s["case"]
    new, total = _lengths(c)
    page, G = c["page"], c["Hq"] // c["Hkv"]
    cu = s["cu_seqlens"].tolist()
    out = torch.zeros(s["T"], c["Hq"], c["D"], dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        n, t = new[b], total[b]
        ids = s["page_table"][b, :_ceil(t, page)].long()
        kk, vv = ((s[x + "_cache"][ids].float().double() * s[x + "_scale"][ids].double()[..., None, None]).transpose(0, 1).reshape(c["Hkv"], -1, c["D"])[:, :t]
                  for x in ("k", "v"))
        pos = t - n + torch.arange(n, device="cuda")
        at = torch.arange(t, device="cuda")
        hide = at[None] > pos[:, None]
        if c["window"]:
            hide |= at[None] <= pos[:, None] - c["window"]
        for h in range(c["Hq"]):
            x = s["q"][cu[b]:cu[b + 1], h].double() @ kk[h // G].t() / math.sqrt(c["D"])
            p = torch.softmax(x.masked_fill(hide, float("-inf")), -1)
            out[cu[b]:cu[b + 1], h] = p @ vv[h // G]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(s["x"])
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        a = _exact_rows(s["x"]) if case["a_form"] == "float" else _exact_held(s["x"], s["x_scales"], M, K)
        y = a @ _exact_held(s["w"], s["w_scales"], N, K).t()
        return y + s["bias"].double() if s["bias"] is not None else y
    return _exact_append(s) if op == "append" else _exact_attention(s)
