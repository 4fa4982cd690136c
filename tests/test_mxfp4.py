"""Microscaled 4-bit floating point: refusals on the CPU; quantisation, layout, values and product on the GPU,
against plain 64-bit restatements (serving_reference)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as R
from xrgpu_b200 import _native

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(cuda_lib):
    from xrgpu_b200 import functional
    return functional


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def _problem(**kw):
    p = _native.Mxfp4Problem_()
    p.dtype, p.a_dtype, p.M, p.K, p.N = _native.FLOAT16, _native.UINT8, 2, 64, 8
    p.a = p.a_scales = p.b = p.b_scales = p.y = 4096
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,message", [
    (dict(dtype=_native.INT8), "T1 must be"),
    (dict(a_dtype=_native.INT8), "activations must be"),
    (dict(M=-1), "geometry"), (dict(K=0), "geometry"), (dict(N=0), "geometry"), (dict(M=1 << 40), "geometry"),
    (dict(ldy=7), "ldy"), (dict(a_dtype=_native.FLOAT16, lda=63), "lda"),
    (dict(a=None), "null"), (dict(y=None), "null"), (dict(b=None), "null"), (dict(b_scales=None), "null"),
    (dict(a_scales=None), "null"), (dict(b=4100), "aligned"), (dict(a=4104), "aligned"), (dict(a_scales=4097), "aligned"),
])
def test_product_refusals(cuda_lib, change, message):
    st = cuda_lib.xrgpu_mxfp4_forward(ctypes.byref(_problem(**change)), None, 0, None)
    assert st == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()


def test_product_refuses_small_workspace(cuda_lib):
    p = _problem(a_dtype=_native.FLOAT16, a_scales=None)
    need = ctypes.c_uint64()
    assert cuda_lib.xrgpu_mxfp4_workspace_size(ctypes.byref(p), ctypes.byref(need)) == 0
    assert need.value == 256 + 512
    assert cuda_lib.xrgpu_mxfp4_forward(ctypes.byref(p), 4096, need.value - 1, None) == _native.INVALID_ARGUMENT
    assert "workspace too small" in cuda_lib.xrgpu_last_error().decode()
    assert cuda_lib.xrgpu_mxfp4_forward(ctypes.byref(p), 4100, need.value, None) == _native.INVALID_ARGUMENT
    p.M = 0
    assert cuda_lib.xrgpu_mxfp4_workspace_size(ctypes.byref(p), ctypes.byref(need)) == 0 and need.value == 0
    assert cuda_lib.xrgpu_mxfp4_forward(ctypes.byref(p), None, 0, None) == 0  # no rows: nothing to do


@pytest.mark.parametrize("change,args,message", [
    (dict(dtype=_native.UINT8), (4096, 0), "T1"), (dict(rows=-1), (4096, 0), "geometry"), (dict(K=0), (4096, 0), "geometry"),
    (dict(), (None, 0), "null"), (dict(), (4096, 31), "ldx"), (dict(codes=4097), (4096, 0), "aligned"),
    (dict(scales=None), (4096, 0), "null"),
])
def test_quantize_refusals(cuda_lib, change, args, message):
    t = _native.Mxfp4Tensor_(_native.FLOAT16, 0, 2, 32, 4096, 4096)
    for k, v in change.items():
        setattr(t, k, v)
    assert cuda_lib.xrgpu_mxfp4_quantize(ctypes.byref(t), *args, None) == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()
    if "ldx" not in message:
        assert cuda_lib.xrgpu_mxfp4_dequantize(ctypes.byref(t), args[0], None) == _native.INVALID_ARGUMENT


def test_python_refusals(F):
    x = torch.zeros(2, 64, dtype=torch.float16)
    b, s = torch.zeros(8, 2, 16, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        F.mxfp4_quantize(x)
    with pytest.raises(ValueError, match="T1"):
        F.mxfp4_quantize(x.to(torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        F.matmul_mxfp4(x, b, s)
    with pytest.raises(ValueError, match="K does not match"):
        F.mxfp4_dequantize(b, s, K=96)
    with pytest.raises(ValueError, match="uint8"):
        F.mxfp4_tile_scales(s.view(1, -1).to(torch.int8))


# ------------------------------------------------------------------------------------------ quantisation
def _values(rows, K, dtype, seed):
    """Normals with outlying columns, zeros, exact borders between codes, and blocks of every magnitude."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.05, 20.0, 1.0)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.5, 0.0, -0.0, -0.25, -5.0])
    m = torch.rand(rows, K, generator=g) < 0.3
    x[m] = borders[torch.randint(0, len(borders), (int(m.sum()),), generator=g)]
    kb = -(-K // 32)
    e = torch.randint(-12, 10, (rows, kb), generator=g).repeat_interleave(32, 1)[:, :K]
    x = torch.ldexp(x, e)
    x[torch.rand(rows, K, generator=g) < 0.05] = 0.0
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 1), (3, 33), (129, 100), (5, 4096), (2, 255), (130, 264), (1, 257)])
def test_quantize_is_exact(F, dtype, rows, K):
    x = _values(rows, K, dtype, rows * 1000 + K)
    if rows * K > 200:
        x[0, 5] = float("inf")
        x[-1, K - 1] = float("nan")
    if rows > 2:
        x[1] = 0.0
    codes, scales, values = R.mx_quantize(x.double().numpy())
    c, s = F.mxfp4_quantize(x.cuda())
    assert np.array_equal(s.cpu().numpy(), R.mx_tile(scales))
    assert np.array_equal(c.cpu().numpy(), codes)
    got = F.mxfp4_dequantize(c, s, K=K).cpu().double().numpy()
    assert np.array_equal(got, values, equal_nan=True)
    assert np.array_equal(F.mxfp4_tile_scales(torch.from_numpy(scales).cuda()).cpu().numpy(), R.mx_tile(scales))


@gpu
def test_quantize_float32_extremes(F):
    """Subnormals, the largest numbers, and what lies under the smallest scale."""
    x = torch.zeros(4, 64)
    x[0, :4] = torch.tensor([3.4028235e38, -1.7e38, 1e38, 1e-45])
    x[1, :4] = torch.tensor([1.1754944e-38, -5.9e-39, 2e-39, 1e-45])
    x[2, :4] = torch.tensor([1e-45, -1e-45, 0.0, 4e-45])
    x[3, 32:36] = torch.tensor([2.0 ** -126, 2.0 ** -125, 2.0 ** -127, 2.0 ** -128])
    codes, scales, values = R.mx_quantize(x.double().numpy())
    c, s = F.mxfp4_quantize(x.cuda())
    assert np.array_equal(c.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), R.mx_tile(scales))
    assert np.array_equal(F.mxfp4_dequantize(c, s).cpu().double().numpy(), values)


@gpu
def test_quantize_strided_rows_and_shapes(F):
    x = torch.randn(6, 7, 200, device="cuda", dtype=torch.float16)
    for view in (x[..., 8:136], x[:, 2:3, :96], x[1:2, 1, 3:103], x[:, 0, 1:]):
        c, s = F.mxfp4_quantize(view)
        c2, s2 = F.mxfp4_quantize(view.contiguous())
        assert c.shape == view.shape[:-1] + (-(-view.shape[-1] // 32), 16)
        assert torch.equal(c, c2) and torch.equal(s, s2)
    with pytest.raises(ValueError, match="one stride"):
        F.mxfp4_quantize(x[:, 1:3, :])
    with pytest.raises(ValueError, match="unit stride"):
        F.mxfp4_quantize(x.transpose(1, 2))
    c, s = F.mxfp4_quantize(x[:0])
    assert c.shape == (0, 7, 7, 16) and s.numel() == 0


# ------------------------------------------------------------------------------------------ product
def _held(rows, K, seed, low=110, high=135):
    g = np.random.default_rng(seed)
    kb = -(-K // 32)
    codes = g.integers(0, 256, (rows, kb, 16), dtype=np.uint8)
    if K % 32:  # padding of the last block is zero codes
        n = np.stack([codes[:, -1] & 15, codes[:, -1] >> 4], -1).reshape(rows, 32)
        n[:, K % 32:] = 0
        codes[:, -1] = n[:, 0::2] | (n[:, 1::2] << 4)
    scales = g.integers(low, high, (rows, kb), dtype=np.uint8)
    return codes, scales


def _bound(a, w, y, dtype, K):
    """Error of float32 sums in steps of at most 32 exact products, each step and each join of partial sums rounded (or
    truncated: 2^-23) relative to the sum of magnitudes, and the result's own rounding."""
    size = np.abs(a) @ np.abs(w).T
    return (K / 32 + 24) * 2.0 ** -23 * size + np.abs(y) * (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24) + 2.0 ** -24 * (dtype == torch.float16)


SHAPES = [(1, 1, 1), (1, 8, 32), (1, 128, 256), (2, 129, 288), (7, 250, 544), (16, 128, 4096), (17, 384, 1024), (33, 1003, 100),
          (64, 256, 1056), (65, 130, 800), (127, 64, 512), (128, 257, 2080), (129, 255, 260), (200, 640, 384), (300, 520, 1312), (1, 4096, 14336),
          (1200, 5900, 544), (1300, 10300, 288), (20, 57001, 64)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(F, dtype, M, N, K):
    lo, hi = (118, 128) if dtype == torch.float16 else (110, 135)  # float16: within its range
    ac, asc = _held(M, K, M + N, lo, hi)
    wc, ws = _held(N, K, K + 1, lo, hi)
    if dtype == torch.float16:
        ws = np.clip(ws, 118, 121)
    bias = torch.randn(N).to(dtype)
    a, w = R.mx_values(ac, asc, K), R.mx_values(wc, ws, K)
    y = a @ w.T
    d = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    args = dict(a_scales=d(R.mx_tile(asc)), K=K, dtype=dtype)
    got = F.matmul_mxfp4(d(ac), d(wc), d(R.mx_tile(ws)), **args)
    assert got.dtype == dtype and got.shape == (M, N)
    assert (np.abs(got.cpu().double().numpy() - y) <= _bound(a, w, y, dtype, K)).all()
    y = y + bias.double().numpy()
    got2 = F.matmul_mxfp4(d(ac), d(wc), d(R.mx_tile(ws)), bias.cuda(), **args)
    assert (np.abs(got2.cpu().double().numpy() - y) <= _bound(a, w, y, dtype, K) + np.abs(bias.double().numpy()) * 2.0 ** -23).all()
    assert torch.equal(got, F.matmul_mxfp4(d(ac), d(wc), d(R.mx_tile(ws)), **args))  # the same bits again


@gpu
@pytest.mark.parametrize("M,N,K", [(3, 70, 100), (40, 200, 512), (150, 300, 320)])
def test_product_of_floats_is_the_quantised_one(F, M, N, K):
    x = torch.randn(M, K, device="cuda", dtype=torch.float16)
    wc, ws = F.mxfp4_quantize(torch.randn(N, K, device="cuda") * 0.1)
    c, s = F.mxfp4_quantize(x)
    want = F.matmul_mxfp4(c, wc, ws, a_scales=s, K=K)
    assert torch.equal(F.matmul_mxfp4(x, wc, ws), want)
    wide = torch.full((M, K + 24), float("nan"), device="cuda", dtype=torch.float16)
    wide[:, 8:8 + K] = x
    assert torch.equal(F.matmul_mxfp4(wide[:, 8:8 + K], wc, ws), want)
    out = torch.full((M, N + 5), 7.0, device="cuda", dtype=torch.float32)
    got = F.matmul_mxfp4(x.view(1, M, K), wc, ws, dtype=torch.float32, out=out[:, 2:2 + N].unsqueeze(0))
    assert got.shape == (1, M, N) and bool((out[:, :2] == 7).all()) and bool((out[:, 2 + N:] == 7).all())
    assert torch.equal(out[:, 2:2 + N].half(), want)


@gpu
@pytest.mark.parametrize("M,N", [(2, 140), (130, 140)])
def test_product_nan_blocks_stay_in_their_rows(F, M, N):
    K = 320
    x, w = torch.randn(M, K), torch.randn(N, K)
    x[1, 40] = float("inf")
    w[133, 300] = float("nan")
    xc, xs = F.mxfp4_quantize(x.cuda())
    wc, ws = F.mxfp4_quantize(w.cuda())
    y = F.matmul_mxfp4(xc, wc, ws, a_scales=xs, K=K, dtype=torch.float32).cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1], bad[:, 133] = True, True
    assert torch.equal(torch.isnan(y), bad)


@gpu
def test_product_wide_scales(F):
    """Scales over the whole range of float32 results: 2^-60 against 2^60, and results that underflow or overflow."""
    K = 64
    ac, _ = _held(4, K, 1)
    wc, _ = _held(8, K, 2)
    asc = np.repeat(np.array([[67], [187], [7], [247]], np.uint8), 2, 1)
    ws = np.repeat(np.array([[67], [187], [127], [7], [247], [100], [127], [154]], np.uint8), 2, 1)
    a, w = R.mx_values(ac, asc, K), R.mx_values(wc, ws, K)
    y = a @ w.T
    d = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    got = F.matmul_mxfp4(d(ac), d(wc), d(R.mx_tile(ws)), a_scales=d(R.mx_tile(asc)), dtype=torch.float32).cpu().double().numpy()
    fits = (np.abs(a) @ np.abs(w).T < 1e38) & (np.abs(y) > 1e-37)
    tol = _bound(a, w, y, torch.float32, K)
    assert fits.sum() >= 20 and (np.abs(got - y)[fits] <= tol[fits]).all()


@gpu
def test_streams_and_graphs(F):
    """Two captured products replay with new inputs, interleaved, on a stream of their own."""
    K, N = 1024, 384
    wc, ws = F.mxfp4_quantize(torch.randn(N, K, device="cuda"))
    xs = [torch.randn(m, K, device="cuda", dtype=torch.float16) for m in (1, 150)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in xs:
            F.matmul_mxfp4(x, wc, ws)
        side.synchronize()
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(F.matmul_mxfp4(x, wc, ws))
            graphs.append(g)
    torch.cuda.synchronize()
    for r in range(3):
        for x in xs:
            x.copy_(torch.randn_like(x))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            assert torch.equal(o, F.matmul_mxfp4(x, wc, ws))


@gpu
def test_refusals_on_device(F):
    x = torch.randn(4, 64, device="cuda", dtype=torch.float16)
    c, s = F.mxfp4_quantize(x)
    with pytest.raises(ValueError, match="differ in K"):
        F.matmul_mxfp4(x[:, :32].contiguous(), c, s)
    with pytest.raises(ValueError, match="tiled scales"):
        F.matmul_mxfp4(x, c, s[:, :0])
    with pytest.raises(ValueError, match="bias"):
        F.matmul_mxfp4(x, c, s, torch.zeros(3, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="out"):
        F.matmul_mxfp4(x, c, s, out=torch.zeros(4, 5, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="CUDA tensor"):
        F.matmul_mxfp4(x, c.cpu(), s)


@pytest.mark.parametrize("a_blocks,b_blocks,rows", [(4, 2, 2), (2, 4, 4), (6, 5, 100)])
@pytest.mark.parametrize("given_k", [False, True])
def test_held_activations_of_another_k_are_refused(F, monkeypatch, a_blocks, b_blocks, rows, given_k):
    """Codes of another number of blocks than the weights': refused on the host, nothing is launched. Their tiled scales'
    shape may well be the one expected, and so may their number of bytes."""
    calls = []
    monkeypatch.setattr(F, "_device_of", lambda t, name: t.get_device())  # tensors on the CPU, as far as the launch
    monkeypatch.setattr(F, "_launch", lambda *args: calls.append(args))
    z = lambda *shape: torch.zeros(*shape, dtype=torch.uint8)  # noqa: E731
    tiles = lambda r, kb: z(-(-r // 128), -(-kb // 4), 32, 4, 4)  # noqa: E731
    K = b_blocks * 32 if given_k else None
    b, b_scales = z(8, b_blocks, 16), tiles(8, b_blocks)
    for scales in (tiles(rows, a_blocks), tiles(rows, b_blocks), tiles(rows * a_blocks // b_blocks, b_blocks)):
        with pytest.raises(ValueError, match="differ in K"):
            F.matmul_mxfp4(z(rows, a_blocks, 16), b, b_scales, a_scales=scales, K=K)
    for shape in ((rows * b_blocks * 16,), (rows, b_blocks * 16), (rows, b_blocks, 8, 2)):
        with pytest.raises(ValueError):
            F.matmul_mxfp4(z(*shape), b, b_scales, a_scales=tiles(rows, b_blocks), K=K)
    assert not calls
    y = F.matmul_mxfp4(z(1, rows, b_blocks, 16), b, b_scales, a_scales=tiles(rows, b_blocks), K=K)
    p = calls[0][2]._obj
    assert y.shape == (1, rows, 8) and (p.M, p.N, p.K) == (rows, 8, b_blocks * 32) and len(calls) == 1


@gpu
@pytest.mark.parametrize("M,N,K", [(1150, 4300, 4130), (1200, 5900, 96), (2240, 9000, 1056), (300, 14000, 8224), (4100, 2300, 2080), (129, 37900, 544)])
def test_product_of_pairs_is_exact_again_and_again(F, M, N, K):
    """Products by pairs of CTAs (whole and halved last rounds, ragged edges, many and few steps along K) whose sums are exact in
    float32, with new operands in the same buffers each time: a tile read before its loads have landed, or
    overwritten before it was read, would show."""
    assert -(-M // 128) * -(-N // 256) > 148
    kb = -(-K // 32)
    g = torch.Generator(device="cuda").manual_seed(M)
    held = []
    for rows in (M, N):
        held += [torch.empty(rows, kb, 16, dtype=torch.uint8, device="cuda"), torch.empty(-(-rows // 128), -(-kb // 4), 32, 4, 4, dtype=torch.uint8, device="cuda")]
    out = torch.empty(M, N, device="cuda")
    for _ in range(6):
        for i, rows in ((0, M), (2, N)):
            x = torch.randint(0, 256, (rows, kb, 16), generator=g, dtype=torch.uint8, device="cuda")
            if K % 32:  # padding of the last block is zero codes
                x[:, -1, K % 32 // 2:] = 0
            held[i].copy_(x)
            held[i + 1].copy_(F.mxfp4_tile_scales(torch.randint(127, 129, (rows, kb), generator=g, dtype=torch.uint8, device="cuda")))
        out.fill_(float("nan"))
        F.matmul_mxfp4(held[0], held[2], held[3], a_scales=held[1], K=K, dtype=torch.float32, out=out)
        a, w = (F.mxfp4_dequantize(held[i], held[i + 1], K=K).double() for i in (0, 2))
        assert torch.equal(out.double(), a @ w.t())  # below 2^24 quarters
    assert F.device_error(0) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(256, 14336, 544), (200, 14200, 96), (129, 18900, 4130), (250, 9700, 2080)])
def test_product_of_single_ctas_with_256_columns(F, dtype, M, N, K):
    """Tiles of 128 x 256 by one CTA each: more tiles of 128 columns than SMs, no more of 256; sums exact in float32."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert M > 128 and -(-M // 128) * -(-N // 128) > sms >= -(-M // 128) * -(-N // 256)
    kb = -(-K // 32)
    g = torch.Generator(device="cuda").manual_seed(M)
    held = []
    for rows in (M, N):
        x = torch.randint(0, 256, (rows, kb, 16), generator=g, dtype=torch.uint8, device="cuda")
        if K % 32:
            x[:, -1, K % 32 // 2:] = 0
        held += [x, F.mxfp4_tile_scales(torch.randint(119, 121, (rows, kb), generator=g, dtype=torch.uint8, device="cuda"))]
    bias = torch.randn(N, generator=g, device="cuda").to(dtype)
    a, w = (F.mxfp4_dequantize(held[i], held[i + 1], K=K).double() for i in (0, 2))
    y = a @ w.t()
    for _ in range(3):
        got = F.matmul_mxfp4(held[0], held[2], held[3], a_scales=held[1], K=K, dtype=dtype)
        assert torch.equal(got, y.to(dtype))
        got = F.matmul_mxfp4(held[0], held[2], held[3], bias, a_scales=held[1], K=K, dtype=dtype)
        assert torch.equal(got, (y.float() + bias.float()).to(dtype))  # one float32 sum, rounded once
    assert F.device_error(0) == 0
