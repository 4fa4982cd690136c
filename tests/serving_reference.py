"""Plain 64-bit restatements of the block-scaled serving operators, on the CPU: what their tests compare with."""
import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def mx_quantize(x):
    """x [rows, K] -> (codes uint8 [rows, kb, 16], scale bytes uint8 [rows, kb], values float64 [rows, K])."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    kb = -(-K // 32)
    codes = np.zeros((rows, kb, 16), np.uint8)
    scales = np.zeros((rows, kb), np.uint8)
    values = np.zeros((rows, kb * 32))
    p = np.zeros((rows, kb * 32))
    p[:, :K] = x
    p = p.reshape(rows, kb, 32)
    for r in range(rows):
        for j in range(kb):
            b = p[r, j]
            if not np.isfinite(b).all():
                scales[r, j] = 255
                values[r, j * 32:j * 32 + 32] = np.nan
                continue
            a = np.abs(b).max()
            E = max(int(np.frexp(a)[1]) - 1 - 2, -127) if a > 0 else -127
            v = np.abs(b) * 2.0 ** -E
            d = np.abs(v[:, None] - E2M1[None])
            near = d == d.min(1, keepdims=True)
            even = np.arange(8) % 2 == 0
            # the nearest code; of two equally near the even one
            c = np.array([next(i for i in sorted(range(8), key=lambda i: (not even[i], i)) if near[n, i]) for n in range(32)])
            c = np.where(v >= 6.0, 7, c)
            values[r, j * 32:j * 32 + 32] = np.where(np.signbit(b), -1.0, 1.0) * E2M1[c] * 2.0 ** E
            c = c + 8 * np.signbit(b)
            codes[r, j] = c[0::2] | (c[1::2] << 4)
            scales[r, j] = E + 127
    return codes, scales, values[:, :K]


def mx_tile(scales):
    rows, kb = scales.shape
    out = np.zeros((-(-rows // 128), -(-kb // 4), 32, 4, 4), np.uint8)
    r, j = np.meshgrid(np.arange(rows), np.arange(kb), indexing="ij")
    out[r // 128, j // 4, r % 32, (r % 128) // 32, j % 4] = scales
    return out


def mx_values(codes, scales, K):
    """float64 [rows, K] of codes [rows, kb, 16] and untiled scale bytes [rows, kb]."""
    rows, kb, _ = codes.shape
    n = np.stack([codes & 15, codes >> 4], -1).reshape(rows, kb, 32).astype(np.int64)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (np.where(n >= 8, -1.0, 1.0) * E2M1[n & 7] * s[..., None]).reshape(rows, kb * 32)[:, :K]


def round_code(x, dtype):
    """float64 -> the nearest code value of the cache's type, ties to even, as float64."""
    L = LIMIT[dtype]
    if dtype == torch.int8:
        return np.clip(np.rint(x), -L, L)
    step = 2.0 ** (np.maximum(np.frexp(x)[1] - 1, -6) - 3)
    return np.clip(np.rint(x / step) * step, -L, L)


class Cache:
    """A paged cache in float64 code values, with the torch tensors that the framework's calls take."""

    def __init__(self, lens, *, heads, D, page, code, seed=0, spare=2, max_extra=1, fill="used"):
        g = torch.Generator().manual_seed(seed)
        self.page, self.heads, self.D, self.code = page, heads, D, code
        need = [-(-max(n, 0) // page) for n in lens]
        P = sum(need) + spare
        order = torch.randperm(P, generator=g).tolist()
        self.table = torch.full((len(lens), max(need + [0]) + max_extra), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.unused = order[at:]
        L = LIMIT[code]

        def side():
            x = torch.randn(P, heads, page, D, generator=g) * (L / 3.5)
            x = x.clamp(-L, L)
            return (x.round().to(torch.int8) if code == torch.int8 else x.to(code)), (torch.rand(P, heads, generator=g) * 1.5 + 0.5) * 3.5 / L

        self.k, self.ks = side()
        self.v, self.vs = side()
        self.lens = torch.tensor(lens, dtype=torch.int32)

    def poison_tails(self, byte=0x7F):
        """Codes behind every sequence's last token (and of unused pages) set to `byte` (0x7f is NaN in e4m3)."""
        for c in (self.k, self.v):
            raw = c.view(torch.uint8)
            for b, n in enumerate(self.lens.tolist()):
                if n % self.page:
                    raw[self.table[b, n // self.page], :, n % self.page:] = byte
            for p in self.unused:
                raw[p] = byte
        for s in (self.ks, self.vs):
            for p in self.unused:
                s[p] = float("nan")

    def cuda(self, device="cuda"):
        return [t.to(device) for t in (self.k, self.v, self.ks, self.vs, self.table)]

    def tokens(self, b, n=None):
        """float64 (k, v) [n, heads, D] of the first n tokens of sequence b."""
        n = int(self.lens[b]) if n is None else n
        out = []
        for c, s in ((self.k, self.ks), (self.v, self.vs)):
            ids = self.table[b, :-(-n // self.page)].long()
            x = c[ids].float().double() * s[ids].double()[..., None, None]
            out.append(x.transpose(1, 2).reshape(-1, self.heads, self.D)[:n].numpy())
        return out


def append(cache, k, v, cu):
    """The append in float64, in place on cache's (CPU) tensors."""
    for x, codes, scale in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        x = x.double().numpy()
        L = LIMIT[cache.code]
        for b, total in enumerate(cache.lens.tolist()):
            n = int(cu[b + 1] - cu[b])
            start = total - n
            for j in range(start // cache.page, -(-total // cache.page)) if n else ():
                lo, hi = max(start, j * cache.page), min(total, (j + 1) * cache.page)
                pid, held = int(cache.table[b, j]), lo - j * cache.page
                for h in range(cache.heads):
                    rows = x[int(cu[b]) + lo - start:int(cu[b]) + hi - start, h]
                    old = np.float32(scale[pid, h].item()) if held else np.float32(0)
                    if not np.isfinite(rows).all() or not np.isfinite(old):
                        scale[pid, h] = float("nan")
                        codes[pid, h, held:held + hi - lo] = 0
                        continue
                    s = max(old, np.float32(np.abs(rows).max()) / np.float32(L))
                    if held and s > old:
                        c = codes[pid, h, :held].float().double().numpy()
                        codes[pid, h, :held] = torch.from_numpy(round_code(c * float(old) / float(s), cache.code)).to(torch.float32).to(cache.code)
                    new = round_code(rows / float(s), cache.code) if s > 0 else np.zeros_like(rows)
                    codes[pid, h, held:held + hi - lo] = torch.from_numpy(new).to(torch.float32).to(cache.code)
                    scale[pid, h] = float(s)


def attention(cache, q, cu, *, scale=None, causal=True, window=0):
    """(o, tolerance) float64 [rows, Hq, D]; rows of no sequence are NaN in o. q: CPU tensor of the call's dtype.

    The tolerance, per value, counts the roundings of a kernel that keeps float32 sums and feeds the
    products with float16 numbers (for float32 rows: pairs of them). With x the scores, p the weights and
    d = (D + 8) 2^-24 max_j sum |scale q k_j| the error of a score (float32 sums over D products):
      weights: exp of a score off by d, 2^-21 of the exponential itself, rounding r of the weight (2^-11 as
      one float16, 2^-21 as a pair), each counted once in the sum of values and once in the normaliser;
      sums over n tokens in float32: n 2^-24 at the very most, taken as (64 + n / 64) 2^-24 (64 tokens a step);
      weights below 2^-14 of the largest lose steps of 2^-25 as float16: 2^-25 of the values' sum;
      the result: 2^-11 or 2^-24 of itself.
    """
    f16 = q.dtype == torch.float16
    T, Hq, D = q.shape
    G = Hq // cache.heads
    scale = D ** -0.5 if scale is None else scale
    o = np.full((T, Hq, D), np.nan)
    tol = np.zeros((T, Hq, D))
    qd = q.double().numpy()
    for b, total in enumerate(cache.lens.tolist()):
        n = int(cu[b + 1] - cu[b])
        k, v = cache.tokens(b)
        for i in range(n):
            pos, row = total - n + i, int(cu[b]) + i
            hi = min(pos + 1, total) if causal else total
            lo = max(0, pos - window + 1) if window else 0
            for h in range(Hq):
                kk, vv = k[lo:max(hi, lo), h // G], v[lo:max(hi, lo), h // G]
                if len(kk) == 0:
                    o[row, h] = 0
                    continue
                x = kk @ qd[row, h] * scale
                w = np.exp(x - x.max())
                p = w / w.sum()
                o[row, h] = p @ vv
                d = (D + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qd[row, h])).max() * abs(scale)
                r = 2.0 ** -11 if f16 else 2.0 ** -21
                size = p @ np.abs(vv)
                rel = 2 * d + 2.0 ** -20 + 2 * r + (64 + len(kk) / 64) * 2.0 ** -24
                tol[row, h] = rel * size + 2.0 ** -25 / w.sum() * np.abs(vv).sum(0) + (2.0 ** -11 if f16 else 2.0 ** -24) * np.abs(o[row, h]) + 2.0 ** -24 * f16
    return o, tol
