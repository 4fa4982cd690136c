"""8-bit integer operators at the ends of their ranges: subnormal scales, scales whose products leave float32 on the way,
empty orders and sums, K split over a cluster, float rows read several times."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import int8_reference as R
from test_int8 import F, FULL, HALF, _codes, _groups, _summed, _values, gpu  # noqa: F401


# ------------------------------------------------------------------------------------------ subnormal scales
def _units(u):
    """Multiples of 2^-149, the smallest float32 step, as they are."""
    u = np.asarray(u, np.int64)
    return torch.from_numpy((np.abs(u) | np.where(u < 0, 1 << 31, 0)).astype(np.uint32).view(np.float32).copy())


@gpu
@pytest.mark.parametrize("K", [5, 8, 100, 9000])
def test_codes_of_subnormal_scales_saturate(F, K):
    """A scale of few bits may lie a third under max|x| / 127: quotients up to 190, also those that leave no remainder. Every
    largest magnitude up to the one where the scale has all its quotients within 127, and beyond."""
    most = 17000 if K < 100 else 700
    u = np.zeros((most, K), np.int64)
    top = np.arange(most)
    for i, v in enumerate((top, -top, top // 2, -(top // 3), top - 1)):
        u[:, (i * 7) % K] = np.where(top > 0, v, 0)
    x = _units(u)
    codes, scales = R.quantize(x.double().numpy())
    c, s = F.int8_quantize(x.cuda())
    assert np.array_equal(s.cpu().double().numpy(), scales) and np.array_equal(c.cpu().numpy(), codes)


@gpu
@pytest.mark.parametrize("M", [12, 40])
def test_products_of_subnormal_rows_saturate(F, M):
    """Rows quantised by the product (12: in the product's own kernel), by weights that pick out one code each."""
    K = 64
    top = np.resize([128, 130, 190, 191, 5000, 127, 254, 71, 317, 1, 63, 64], M)
    u = np.zeros((M, K), np.int64)
    u[:, 0], u[:, 1], u[:, 9], u[:, 40] = top, -top, top // 2, -(top // 4)
    x = _units(u)
    codes, scales = R.quantize(x.double().numpy())
    w = torch.eye(K, dtype=torch.int8, device="cuda")
    y = F.matmul_int8(x.cuda(), w, torch.full((K,), 2.0 ** 40, device="cuda"))
    assert np.array_equal(y.cpu().double().numpy(), codes * scales[:, None] * 2.0 ** 40)  # a code by a scale of few bits: exact


# ------------------------------------------------------------------------------------------ scales far apart
def _far_scales(g, M, N):
    """Rows of ordinary scales, of ones whose product with a sum leaves float32, and channels that bring it back."""
    sa = torch.exp2(torch.randint(-20, 6, (M,), generator=g).float())
    far = torch.rand(M, generator=g) < 0.5
    sa[far] = torch.exp2(96 + 31 * torch.rand(int(far.sum()), generator=g))
    sa[0] = 2.0 ** 127
    sign = lambda n: torch.where(torch.rand(n, generator=g) < 0.2, -1.0, 1.0)  # noqa: E731
    return sa * sign(M), torch.exp2(-100 - 20 * torch.rand(N, generator=g)) * sign(N)


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 130, 4096), (40, 130, 70), (16, 4096, 2048), (333, 1004, 1100), (700, 5000, 300), (2300, 3000, 1057)])
@pytest.mark.parametrize("act,bias", [("none", False), ("relu", True), ("swiglu", True)])
def test_scales_far_apart(F, M, N, K, act, bias):
    g = torch.Generator().manual_seed(M + K)
    a, ad, _ = _codes(g, M, K)
    b, bd, _ = _codes(g, N, K)
    if M > 3:
        a[3], ad[3] = 0, 0
    sa, sb = _far_scales(g, M, N)
    v = torch.randn(N, generator=g) if bias else None
    want, err = R.product(a, sa.double().numpy(), b, sb.double().numpy(), v.double().numpy() if bias else None, act)
    y = F.matmul_int8(ad, bd, sb.cuda(), v.cuda() if bias else None, a_scales=sa.cuda(), activation=act, dtype=FULL)
    R.close(y, want, err, FULL)


@gpu
@pytest.mark.parametrize("M,N,K", [(3, 256, 1024), (16, 2000, 600), (50, 200, 1000)])
def test_float_rows_of_large_numbers(F, M, N, K):
    g = torch.Generator().manual_seed(M)
    x = torch.rand(M, K, generator=g) * 3e38
    x[1] *= 2.0 ** -120
    b, bd, _ = _codes(g, N, K)
    sb = torch.rand(N, generator=g) * 2.0 ** -60
    a, sa = R.quantize(x.double().numpy())
    want, err = R.product(a, sa, b, sb.double().numpy())
    R.close(F.matmul_int8(x.cuda(), bd, sb.cuda()), want, err, FULL)


@gpu
def test_grouped_rows_of_large_scales(F):
    g = torch.Generator().manual_seed(2)
    E, rows, N, K, k = 5, 300, 150, 200, 3
    a, ad, _ = _codes(g, rows, K)
    b, bd, _ = _codes(g, E * N, K)
    sa, sb = _far_scales(g, rows, E * N)
    off = _groups(E, rows, 1, "ragged")
    want, err = np.zeros((rows, N)), np.zeros((rows, N))
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            want[lo:hi], err[lo:hi] = R.product(a[lo:hi], sa[lo:hi].double().numpy(), b.reshape(E, N, K)[e], sb.view(E, N)[e].double().numpy())
    args = (ad, bd.unflatten(0, (E, N)), sb.view(E, N).cuda(), torch.from_numpy(off).int().cuda())
    kw = dict(a_scales=sa.cuda(), dtype=FULL)
    R.close(F.matmul_int8_grouped(*args, **kw), want, err, FULL)
    slots = torch.randperm(rows, generator=g).view(-1, k)
    weights = torch.rand(slots.shape, generator=g)
    y = F.matmul_int8_grouped(*args, **kw, slots=slots.int().cuda(), weights=weights.cuda())
    R.close(y, *_summed(want, err, slots.numpy(), weights.numpy()), FULL)


# ------------------------------------------------------------------------------------------ K split over a cluster
@gpu
@pytest.mark.parametrize("M", [20, 40, 67, 75, 90, 107, 128, 139, 155, 250])
@pytest.mark.parametrize("N,K", [(130, 4096), (1000, 2050)])
def test_split_products_of_every_width(F, M, N, K):
    g = torch.Generator().manual_seed(M + N)
    a, ad, sa = _codes(g, M, K)
    b, bd, sb = _codes(g, N, K)
    want, err = R.product(a, sa.double().numpy(), b, sb.double().numpy())
    R.close(F.matmul_int8(ad, bd, sb.cuda(), a_scales=sa.cuda(), dtype=FULL), want, err, FULL)
    assert F.device_error() == 0


# ------------------------------------------------------------------------------------------ nothing to do
@gpu
@pytest.mark.parametrize("floats", [True, False])
def test_no_rows_of_some_tokens(F, floats):
    """Tokens of which none chose one of these experts, and sums for no tokens."""
    w, ws = F.int8_quantize(torch.ones(4, 48, 64, device="cuda"))
    x, kw = torch.ones(6, 64, device="cuda"), dict(dtype=FULL)
    if not floats:
        x, kw["a_scales"] = F.int8_quantize(x)
    off = torch.zeros(5, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert F.matmul_int8_grouped(x, w, ws, off, order=none, top_k=2, **kw).shape == (0, 48)
    slots, weights = torch.full((6, 2), -1, dtype=torch.int32, device="cuda"), torch.ones(6, 2, device="cuda")
    y = F.matmul_int8_grouped(x, w, ws, off, order=none, top_k=2, slots=slots, weights=weights, **kw)
    assert y.shape == (6, 48) and (y == 0).all()
    off[1:] = 6
    assert F.matmul_int8_grouped(x, w, ws, off, slots=slots[:0], weights=weights[:0], **kw).shape == (0, 48)
    out = torch.full((3, 48), 5.0, device="cuda")
    assert F.matmul_int8_grouped(x, w, ws, off, slots=slots[:0], weights=weights[:0], out=out[:0], **kw).shape == (0, 48)
    assert (out == 5).all() and F.device_error() == 0


# ------------------------------------------------------------------------------------------ float rows read several times
@gpu
@pytest.mark.parametrize("T,E,k,N,K", [(1100, 7, 4, 130, 2048), (1100, 5, 4, 66, 2050), (1000, 9, 4, 96, 2050), (300, 3, 32, 64, 1000)])
@pytest.mark.parametrize("dtype,act", [(HALF, "swiglu"), (FULL, "none")])
def test_float_tokens_read_several_times(F, dtype, act, T, E, k, N, K):
    """Gathered float rows on both sides of the size from which tokens are quantised once: strided, in turn with new ones, entries
    that fit no row among them, as rows and as sums."""
    rng = np.random.default_rng(T + K)
    rows = T * k
    g = torch.Generator().manual_seed(K)
    b, bd, sb = _codes(g, E * N, K)
    bd, sb = bd.unflatten(0, (E, N)), (sb / K ** 0.5).view(E, N)
    wide = torch.zeros(T, K + 13, dtype=dtype, device="cuda")
    slots, weights = rng.permutation(rows).reshape(T, k), rng.normal(size=(T, k)).astype(np.float32)
    sums = dict(slots=torch.from_numpy(slots).int().cuda(), weights=torch.from_numpy(weights).cuda())
    calls = []
    for turn, lead in enumerate((0, 8, 3)):
        x = _values(T, K, dtype, turn + K)
        x[5], x[6, K - 1] = 0.0, float("nan")
        order = rng.permutation(rows) if turn else np.repeat(rng.permutation(T), k) * k
        if turn == 2:
            order[[0, 7, rows - 1]] = [-1, rows, 2 ** 31 - 1]
        off = _groups(E, rows, turn, "ragged")
        wide[:, lead:lead + K].copy_(x)
        args = (wide[:, lead:lead + K], bd, sb.cuda(), torch.from_numpy(off).int().cuda())
        kw = dict(order=torch.from_numpy(order).int().cuda(), top_k=k, activation=act)
        calls.append((x, order, off, F.matmul_int8_grouped(*args, **kw), F.matmul_int8_grouped(*args, **kw, **sums)))
    assert F.device_error() == 0x702
    for x, order, off, y, s in calls:
        codes, scales = R.quantize(x.double().numpy())
        fits = (order >= 0) & (order < rows)
        token = np.where(fits, order // k, 0)
        a, sa = np.where(fits[:, None], codes[token], 0), np.where(fits, scales[token], 0.0)
        want, err = np.zeros((rows, N // 2 if act == "swiglu" else N)), np.zeros((rows, N // 2 if act == "swiglu" else N))
        for e in range(E):
            lo, hi = off[e], off[e + 1]
            if lo < hi:
                want[lo:hi], err[lo:hi] = R.product(a[lo:hi], np.nan_to_num(sa[lo:hi]), b.reshape(E, N, K)[e], sb[e].double().numpy(), None, act)
        want[np.isnan(sa)] = np.nan
        R.close(y, want, err, dtype)
        R.close(s, *_summed(want, err, slots, weights), dtype)


@gpu
def test_captured_tokens_read_several_times(F):
    """The chain of quantisation, copies and product in a graph, replayed with new tokens and another order."""
    g = torch.Generator().manual_seed(1)
    T, E, k, N, K = 1100, 6, 4, 128, 2048
    w, ws = F.int8_quantize(torch.randn(E, N, K, generator=g).cuda())
    x, scores = torch.randn(T, K, generator=g, dtype=HALF).cuda(), torch.randn(T, E, generator=g).cuda()

    def layer():
        r = F.moe_route(scores, k)
        return F.matmul_int8_grouped(x, w, ws, r.offsets, order=r.order, top_k=k, slots=r.slots, weights=r.weights)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer()
    for turn in range(4):
        x.copy_(torch.randn(T, K, generator=g, dtype=HALF))
        scores.copy_(torch.randn(T, E, generator=g))
        graph.replay()
        assert torch.equal(y, layer())
    assert F.device_error() == 0
