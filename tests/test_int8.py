"""8-bit integer rows and products, dense and grouped, and the expert router: refusals on the CPU; codes, values, choices
and products on the GPU, against plain 64-bit restatements (int8_reference)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import int8_reference as R
from xrgpu_b200 import _native

gpu = pytest.mark.gpu
HALF, FULL = torch.float16, torch.float32


@pytest.fixture(scope="module")
def F(cuda_lib):
    from xrgpu_b200 import functional
    return functional


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def _problem(**kw):
    p = _native.Int8Problem_()
    p.dtype, p.a_dtype, p.M, p.K, p.N = _native.FLOAT16, _native.INT8, 2, 64, 8
    p.alpha = 1.0
    p.a = p.a_scales = p.b = p.b_scales = p.y = 4096
    for k, v in kw.items():
        setattr(p, k, v)
    return p


GROUPED = dict(groups=4, rows=6, M=6, offsets=4096)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=_native.INT8), "T1 must be"), (dict(a_dtype=_native.UINT8), "activations must be"),
    (dict(M=-1), "geometry"), (dict(K=0), "geometry"), (dict(K=131072), "geometry"), (dict(N=0), "geometry"),
    (dict(N=1 << 40), "geometry"), (dict(M=1 << 40), "geometry"), (dict(groups=-1), "geometry"),
    (dict(**{**GROUPED, "groups": 1025}), "geometry"), (dict(**{**GROUPED, "N": 1 << 29}), "geometry"),
    (dict(activation=_native.ACT_GELU), "activation"), (dict(activation=_native.ACT_SWIGLU, N=7), "pairs"),
    (dict(activation=_native.ACT_SWIGLU, alpha=float("nan")), "finite"),
    (dict(activation=_native.ACT_SWIGLU, has_limit=1, limit=-1.0), "limit"),
    (dict(lda=72), "16 bytes"), (dict(lda=48), "16 bytes"), (dict(ldb=65), "16 bytes"),
    (dict(a_dtype=_native.FLOAT16, lda=63), "lda"), (dict(ldy=7), "ldy"), (dict(activation=_native.ACT_SWIGLU, ldy=3), "ldy"),
    (dict(a=None), "null"), (dict(a_scales=None), "null"), (dict(b=None), "null"), (dict(b_scales=None), "null"), (dict(y=None), "null"),
    (dict(b=4104), "aligned"), (dict(a=4097), "aligned"), (dict(offsets=4096), "dense"), (dict(order=4096), "dense"),
    (dict(**{**GROUPED, "offsets": None}), "null"), (dict(**{**GROUPED, "rows": 5}), "product's rows"),
    (dict(**{**GROUPED, "rows": -1}), "geometry"), (dict(**{**GROUPED, "order": 4096}), "top_k"),
    (dict(**{**GROUPED, "order": 4096, "top_k": 1, "M": 0}), "rows of a"),
    (dict(**{**GROUPED, "slots": 4096, "top_k": 2, "tokens": 3}), "belong together"),
    (dict(**{**GROUPED, "weights": 4096}), "belong together"),
    (dict(**{**GROUPED, "slots": 4096, "weights": 4096, "tokens": 3}), "top_k"),
    (dict(**{**GROUPED, "slots": 4096, "weights": 4096, "tokens": 1 << 30, "top_k": 4}), "geometry"),
])
def test_product_refusals(cuda_lib, change, message):
    st = cuda_lib.xrgpu_int8_forward(ctypes.byref(_problem(**change)), None, 0, None)
    assert st == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()


def test_product_workspace(cuda_lib):
    need = ctypes.c_uint64()
    size = lambda **kw: (cuda_lib.xrgpu_int8_workspace_size(ctypes.byref(_problem(**kw)), ctypes.byref(need)), need.value)  # noqa: E731
    assert size() == (0, 0)
    assert size(a_dtype=_native.FLOAT16) == (0, 0)  # few rows are quantised in place
    assert size(a_dtype=_native.FLOAT16, M=17) == (0, 1280 + 256)  # codes, scales
    assert size(**GROUPED, order=4096, top_k=1) == (0, 512 + 256)  # rows in the groups' order
    assert size(**GROUPED, slots=4096, weights=4096, tokens=3, top_k=2) == (0, 6 * 8 * 4)
    p = _problem(a_dtype=_native.FLOAT16, M=17)
    assert cuda_lib.xrgpu_int8_forward(ctypes.byref(p), 4096, 1535, None) == _native.INVALID_ARGUMENT
    assert "workspace too small" in cuda_lib.xrgpu_last_error().decode()
    assert cuda_lib.xrgpu_int8_forward(ctypes.byref(p), 4100, 1536, None) == _native.INVALID_ARGUMENT
    assert cuda_lib.xrgpu_int8_forward(ctypes.byref(_problem(M=0)), None, 0, None) == 0  # no rows: nothing to do
    assert cuda_lib.xrgpu_int8_forward(None, None, 0, None) == _native.INVALID_ARGUMENT


@pytest.mark.parametrize("change,args,message", [
    (dict(dtype=_native.INT8), (4096, 0), "T1"), (dict(rows=-1), (4096, 0), "geometry"), (dict(K=0), (4096, 0), "geometry"),
    (dict(ldc=40), (4096, 0), "16 bytes"), (dict(ldc=16), (4096, 0), "16 bytes"), (dict(), (None, 0), "null"),
    (dict(), (4096, 31), "ldx"), (dict(codes=4097), (4096, 0), "aligned"), (dict(scales=None), (4096, 0), "null"),
])
def test_quantize_refusals(cuda_lib, change, args, message):
    t = _native.Int8Tensor_(_native.FLOAT16, 0, 2, 32, 0, 4096, 4096)
    for k, v in change.items():
        setattr(t, k, v)
    assert cuda_lib.xrgpu_int8_quantize(ctypes.byref(t), *args, None) == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()
    if "ldx" not in message:
        assert cuda_lib.xrgpu_int8_dequantize(ctypes.byref(t), args[0], None) == _native.INVALID_ARGUMENT


@pytest.mark.parametrize("change,message", [
    (dict(dtype=_native.INT8), "T1"), (dict(experts=0), "router"), (dict(experts=1025), "router"), (dict(top_k=0), "router"),
    (dict(top_k=9), "router"), (dict(experts=64, top_k=33), "router"), (dict(tokens=-1), "geometry"), (dict(tokens=1 << 40), "geometry"),
    (dict(lds=7), "strides"), (dict(scores=None), "null"), (dict(offsets=None), "null"), (dict(slots=None), "null"),
])
def test_route_refusals(cuda_lib, change, message):
    p = _native.MoeRouteProblem_(_native.FLOAT16, 1, 3, 8, 2, 0, 4096, 4096, 4096, 4096, 4096, 4096)
    for k, v in change.items():
        setattr(p, k, v)
    assert cuda_lib.xrgpu_moe_route(ctypes.byref(p), None, 0, None) == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()


def test_python_refusals(F):
    x = torch.zeros(2, 64, dtype=HALF)
    w, s = torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(ValueError, match="T1"):
        F.int8_quantize(x.to(torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        F.int8_quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        F.int8_dequantize(w, s)
    with pytest.raises(ValueError, match="CUDA"):
        F.matmul_int8(x, w, s)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        F.matmul_int8(x, w[None], s[None])
    with pytest.raises(ValueError, match=r"\[experts, N, K\]"):
        F.matmul_int8_grouped(x, w, s, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="T1"):
        F.moe_route(torch.zeros(2, 8, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="CUDA"):
        F.moe_route(torch.zeros(2, 8), 2)


@gpu
def test_python_refusals_of_device_tensors(F):
    x = torch.zeros(2, 40, dtype=HALF, device="cuda")
    w, s = F.int8_quantize(torch.ones(8, 40, device="cuda"))
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    w2, s2 = w.expand(2, 8, 40).contiguous(), s.expand(2, 8).contiguous()
    for match, call in [
        ("16-byte", lambda: F.matmul_int8(x, w.contiguous(), s)),            # rows 40 bytes apart
        ("16-byte", lambda: F.matmul_int8(x[:, 1:], w[:, 1:], s)),
        ("differ in K", lambda: F.matmul_int8(x[:, :32], w, s)),
        ("b_scales", lambda: F.matmul_int8(x, w, s[:7])),
        ("b_scales", lambda: F.matmul_int8(x, w, s.half())),
        ("bias", lambda: F.matmul_int8(x, w, s, s)),                          # float32 bias, float16 result
        ("need a_scales", lambda: F.matmul_int8(w, w, s)),
        ("a_scales", lambda: F.matmul_int8(w, w, s, a_scales=s[:2])),
        ("activation", lambda: F.matmul_int8(x, w, s, activation="gelu")),
        ("pairs", lambda: F.matmul_int8(x, w[:7], s[:7], activation="swiglu")),
        ("out must be", lambda: F.matmul_int8(x, w, s, out=x)),
        ("unit stride", lambda: F.matmul_int8(x.t().contiguous().t(), w, s)),
        ("offsets", lambda: F.matmul_int8_grouped(x, F.int8_quantize(torch.ones(2, 8, 40, device="cuda"))[0], s2, off[:2])),
        ("16-byte", lambda: F.matmul_int8_grouped(x, w2, s2, off)),
        ("router", lambda: F.moe_route(x, 41)), ("router", lambda: F.moe_route(x, 33)), ("router", lambda: F.moe_route(x, 0)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    b2 = F.int8_quantize(torch.ones(2, 8, 40, device="cuda"))[0]
    order = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="belong together"):
        F.matmul_int8_grouped(x, b2, s2, off, slots=order.view(2, 2))
    with pytest.raises(ValueError, match="top_k"):
        F.matmul_int8_grouped(x, b2, s2, off, order=order, top_k=4, slots=order.view(2, 2), weights=torch.ones(2, 2, device="cuda"))
    with pytest.raises(ValueError, match="top_k"):
        F.matmul_int8_grouped(x, b2, s2, off, order=order, top_k=0)


# ------------------------------------------------------------------------------------------ rows
def _values(rows, K, dtype, seed):
    """Normals with outlying columns, exact borders between codes, zeros, rows of every magnitude."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.02, 12.0, 1.0)
    m = torch.rand(rows, K, generator=g) < 0.3
    x[m] = (torch.randint(-255, 256, (int(m.sum()),), generator=g) * 0.5).clamp(-127, 127)  # where 127 is the largest: ties
    x[:, K // 2] = torch.where(torch.rand(rows, generator=g) < 0.5, 127.0, x[:, K // 2])
    x = torch.ldexp(x, torch.randint(-12, 6, (rows, 1), generator=g))
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [HALF, FULL])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 4096), (3, 15), (17, 16), (70, 33), (2, 4100), (5, 8192), (3, 16384), (2, 28672), (2, 40000), (300, 64), (33, 250), (700, 1024), (1500, 4096), (1000, 5000), (600, 9008), (650, 24000), (593, 6000), (3000, 9000), (5000, 1024), (2500, 14336)])
def test_quantize_is_exact(F, dtype, rows, K):
    x = _values(rows, K, dtype, rows * 1000 + K)
    if rows > 2:
        x[1] = 0.0
        x[2, K // 3] = float("inf")
        x[-1, K - 1] = float("nan") if rows > 3 else float("-inf")
    codes, scales = R.quantize(x.double().numpy())
    c, s = F.int8_quantize(x.cuda())
    assert c.shape == (rows, K) and c.stride(0) % 16 == 0 and s.shape == (rows,)
    assert np.array_equal(s.cpu().double().numpy(), scales, equal_nan=True)
    assert np.array_equal(c.cpu().numpy(), codes)
    for out in (HALF, FULL):
        want = (torch.from_numpy(codes).float() * torch.from_numpy(scales).float()[:, None]).to(out)
        assert torch.equal(torch.nan_to_num(F.int8_dequantize(c, s, dtype=out).cpu(), nan=123.0), torch.nan_to_num(want, nan=123.0))


@gpu
def test_quantize_float32_extremes(F):
    """The largest numbers, subnormals, scales that underflow, and neighbours of borders one step away."""
    x = torch.zeros(7, 64)
    x[0, :4] = torch.tensor([3.4028235e38, -1.7e38, 1e38, 1e-45])
    x[1, :4] = torch.tensor([1.1754944e-38, -5.9e-39, 2e-39, 1e-45])
    x[2, :4] = torch.tensor([1e-45, -1e-45, 0.0, 4e-45])       # the scale underflows to zero
    x[3, :4] = torch.tensor([1e-43, -1e-43, 5e-44, 1.4e-45])   # a scale of one subnormal step: codes saturate
    x[4, :3] = torch.tensor([1e-30, 3.9370e-33, -5e-31])
    for r, top in ((5, 1.7), (6, 100.3)):
        s = np.float32(top) / np.float32(127)
        border = (np.arange(31) + 0.5).astype(np.float32) * s
        x[r, 0] = top
        x[r, 1:32] = torch.from_numpy(np.nextafter(border, np.float32(0)))
        x[r, 32:63] = torch.from_numpy(-np.nextafter(border, np.float32(1e9)))
    codes, scales = R.quantize(x.double().numpy())
    c, s = F.int8_quantize(x.cuda())
    assert np.array_equal(s.cpu().double().numpy(), scales) and np.array_equal(c.cpu().numpy(), codes)


@gpu
def test_quantize_strided_rows_and_shapes(F):
    x = torch.randn(6, 7, 200, device="cuda", dtype=HALF)
    for view in (x[..., 8:136], x[:, 2:3, :96], x[1:2, 1, 3:103], x[:, 0, 1:], x[:0], x[0, 0]):
        c, s = F.int8_quantize(view)
        assert c.shape == view.shape and s.shape == view.shape[:-1]
        if view.numel():
            codes, scales = R.quantize(view.reshape(-1, view.shape[-1]).cpu().double().numpy())
            assert np.array_equal(c.cpu().numpy().reshape(codes.shape), codes) and np.array_equal(s.cpu().double().numpy().reshape(-1), scales)
    with pytest.raises(ValueError, match="one stride"):
        F.int8_quantize(x[:4, :3].transpose(0, 1))


# ------------------------------------------------------------------------------------------ dense products
def _codes(g, rows, K):
    c = torch.randint(-128, 128, (rows, K), generator=g, dtype=torch.int8)
    held = torch.full((rows, -(-K // 16) * 16), 77, dtype=torch.int8, device="cuda")  # what lies behind a row is not read
    held[:, :K] = c.cuda()
    return c.numpy(), held[:, :K], torch.rand(rows, generator=g) * 0.02 + 0.001


SIZES = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 7, 15), (16, 129, 33), (17, 1003, 4100), (33, 2, 127), (64, 640, 2048), (128, 256, 129),
         (129, 300, 31), (200, 128, 16), (255, 513, 256), (257, 1000, 300), (300, 2049, 128), (1000, 384, 100), (700, 5000, 64), (2049, 700, 257), (2300, 3000, 200), (1030, 9002, 128), (5000, 1500, 96),
         (2048, 5000, 100), (1600, 6500, 700), (4000, 2600, 1300), (260, 15000, 515), (3100, 11000, 140),
         (2300, 3001, 1057), (260, 15000, 1100), (1030, 9002, 1130), (530, 7000, 1025), (9000, 4000, 96)]


@gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype,bias,act", [(HALF, False, "none"), (FULL, True, "none"), (HALF, True, "relu"), (FULL, False, "swiglu"), (HALF, True, "swiglu")])
def test_product_of_codes(F, M, N, K, dtype, bias, act):
    if act == "swiglu":
        N += N % 2
    g = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    a, ad, sa = _codes(g, M, K)
    b, bd, sb = _codes(g, N, K)
    sb = sb / K ** 0.5
    v = torch.randn(N, generator=g).to(dtype) if bias else None
    y = F.matmul_int8(ad, bd, sb.cuda(), v.cuda() if bias else None, a_scales=sa.cuda(), activation=act, dtype=dtype)
    want, err = R.product(a, sa.double().numpy(), b, sb.double().numpy(), v.double().numpy() if bias else None, act)
    R.close(y, want, err, dtype)
    assert F.device_error() == 0


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (5, 100, 70), (16, 4096, 14336), (333, 1003, 4100), (600, 6000, 520)])
@pytest.mark.parametrize("dtype", [HALF, FULL])
def test_product_quantises_floats(F, M, N, K, dtype):
    g = torch.Generator().manual_seed(K)
    x = _values(M, K, dtype, K)
    b, bd, sb = _codes(g, N, K)
    a, sa = R.quantize(x.double().numpy())
    want, err = R.product(a, sa, b, sb.double().numpy())
    R.close(F.matmul_int8(x.cuda(), bd, sb.cuda()), want, err, dtype)
    R.close(F.matmul_int8(x.cuda(), bd, sb.cuda(), dtype=FULL), want, err, FULL)


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (2, 130, 33), (16, 2000, 600), (7, 14336, 1000), (3, 256, 9001), (1, 4096, 4096), (13, 700, 28672), (16, 24000, 100), (4, 29000, 520)])
@pytest.mark.parametrize("dtype,out,act", [(HALF, HALF, "none"), (FULL, FULL, "swiglu"), (HALF, FULL, "relu"), (FULL, HALF, "none")])
def test_product_of_few_float_rows(F, M, N, K, dtype, out, act):
    """Rows that the product's own kernel quantises: strided, with zeros, NaN, infinities and tiny numbers among them."""
    N += N % 2 if act == "swiglu" else 0
    g = torch.Generator().manual_seed(M * N + K)
    x = _values(M, K, dtype, K + M)
    if M > 4:
        x[0], x[1, K // 2], x[2, -1] = 0.0, float("nan"), float("-inf")
        x[3] *= 2.0 ** -120 if dtype == FULL else 2.0 ** -13
    b, bd, sb = _codes(g, N, K)
    v = torch.randn(N, generator=g).to(out)
    a, sa = R.quantize(x.double().numpy())
    want, err = R.product(a, np.nan_to_num(sa), b, sb.double().numpy(), v.double().numpy(), act)
    want[np.isnan(sa)] = np.nan
    wide = torch.randn(M, K + 24, generator=g).to(dtype).cuda()
    for lead in (8, 3):  # rows on 16 bytes (for some K), and rows that are not
        view = wide[:, lead:lead + K]
        view.copy_(x)
        R.close(F.matmul_int8(view, bd, sb.cuda(), v.cuda(), activation=act, dtype=out), want, err, out)
    assert F.device_error() == 0


@gpu
def test_product_sums_are_exact(F):
    """The longest rows at the largest codes: -128 * -128 * 131071 is 2^31 - 2^14; and sums that cancel."""
    K = 131071
    a = torch.full((2, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b = torch.full((3, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b[1] = 127
    b[2, ::2] = 127
    one = torch.ones(3, device="cuda")
    want = (a.cpu().long() @ b.cpu().long().t()).double().numpy()
    y = F.matmul_int8(a, b, one, a_scales=one[:2], dtype=FULL)
    assert np.array_equal(y.cpu().double().numpy(), want.astype(np.float32).astype(np.float64))


@gpu
def test_product_nan_rows_zero_rows_and_limits(F):
    g = torch.Generator().manual_seed(3)
    x = _values(40, 96, FULL, 9) * 10
    x[3, 5], x[7], x[9, 0] = float("nan"), 0.0, float("inf")
    b, bd, sb = _codes(g, 64, 96)
    a, sa = R.quantize(x.double().numpy())
    for act, kw in (("none", {}), ("relu", {}), ("swiglu", dict(alpha=1.7, beta=1.0, limit=2.5)), ("swiglu", dict(limit=0.0))):
        want, err = R.product(a, np.nan_to_num(sa), b, sb.double().numpy(), None, act, **kw)
        want[[3, 9]] = np.nan
        R.close(F.matmul_int8(x.cuda(), bd, sb.cuda(), activation=act, **kw), want, np.nan_to_num(err), FULL)


@gpu
def test_product_strides_and_shapes(F):
    g = torch.Generator().manual_seed(4)
    b, bd, sb = _codes(g, 50, 80)
    x = torch.randn(3, 4, 200, generator=g, dtype=HALF).cuda()
    view = x[..., 7:87]
    a, sa = R.quantize(view.reshape(12, 80).cpu().double().numpy())
    want, err = R.product(a, sa, b, sb.double().numpy())
    y = F.matmul_int8(view, bd, sb.cuda())
    assert y.shape == (3, 4, 50)
    R.close(y.view(12, 50), want, err, HALF)
    for lead in (0, 1, 3):  # columns of a wider result, at even and odd places
        wide = torch.full((3, 4, 61), 5.0, dtype=HALF, device="cuda")
        F.matmul_int8(view, bd, sb.cuda(), out=wide[..., lead:lead + 50])
        assert torch.equal(wide[..., lead:lead + 50], y) and (wide[..., :lead] == 5).all() and (wide[..., lead + 50:] == 5).all()
    both = torch.zeros(100, 160, dtype=torch.int8, device="cuda")  # codes inside a larger matrix
    both[::2, 32:112] = bd
    c, cs = F.int8_quantize(view)
    assert torch.equal(F.matmul_int8(c, both[::2, 32:112], sb.cuda(), a_scales=cs), y)
    assert torch.equal(F.matmul_int8(view[0, 0], bd, sb.cuda()), y[0, 0])
    assert F.matmul_int8(view[:0], bd, sb.cuda()).shape == (0, 4, 50)


# ------------------------------------------------------------------------------------------ router
def _scores(T, E, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * 3
    x[torch.rand(T, E, generator=g) < 0.2] = 1.5  # ties
    x[torch.rand(T, E, generator=g) < 0.05] = float("-inf")
    x[torch.rand(T, E, generator=g) < 0.02] = float("nan")
    if T > 2:
        x[T // 2] = float("-inf")
        x[T - 1] = torch.where(torch.rand(E, generator=g) < 0.5, 0.0, -0.0)
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [HALF, FULL])
@pytest.mark.parametrize("T,E,k,normalize", [(1, 1, 1, True), (1, 64, 8, True), (5, 8, 8, False), (33, 60, 6, True), (64, 128, 8, True), (65, 128, 8, False),
                                             (100, 33, 1, True), (1000, 256, 8, True), (3000, 16, 2, False), (5000, 384, 6, True), (130, 1024, 32, False), (4800, 700, 3, True)])
def test_route(F, dtype, T, E, k, normalize):
    x = _scores(T, E, dtype, T + E)
    experts, weights, order, slots, offsets, bound = R.route(x.double().numpy(), k, normalize)
    r = F.moe_route(x.cuda(), k, normalize=normalize)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    assert np.array_equal(r.order.cpu().numpy(), order) and np.array_equal(r.slots.cpu().numpy(), slots)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    R.close(r.weights, weights, weights * bound, FULL)


@gpu
@pytest.mark.parametrize("dtype", [HALF, FULL])
@pytest.mark.parametrize("E,k", [(32, 32), (64, 8), (128, 32), (160, 32), (200, 7), (256, 8), (256, 32), (512, 16), (999, 32), (1024, 8)])
def test_route_of_distinct_and_nearly_equal_scores(F, dtype, E, k):
    """Distinct scores; favourites at every 32nd place; neighbours one step apart around the k-th; all of this in one call."""
    g = torch.Generator().manual_seed(E + k)
    x = torch.randn(400, E, generator=g).to(dtype)
    for t in range(100, 200):  # the best of all share a place modulo 32
        at = torch.arange(t % 32, E, 32)
        x[t, at] = (10 + torch.randn(len(at), generator=g)).to(dtype)
    for t in range(200, 300):  # the k-th and the next one step apart, the later one the higher
        rank = torch.argsort(-x[t].double(), stable=True)
        if k < E:
            i, j = sorted((int(rank[k - 1]), int(rank[k])))
            v = x[t, rank[k - 1]]
            x[t, i], x[t, j] = v, torch.nextafter(v, torch.tensor(float("inf"), dtype=dtype))
    for t in range(300, 400):  # many within a few steps of one value
        x[t] = (1 + torch.randint(0, 40, (E,), generator=g) * torch.finfo(dtype).eps).to(dtype)
    experts, weights, order, slots, offsets, bound = R.route(x.double().numpy(), k)
    r = F.moe_route(x.cuda(), k)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    assert np.array_equal(r.order.cpu().numpy(), order) and np.array_equal(r.slots.cpu().numpy(), slots) and np.array_equal(r.offsets.cpu().numpy(), offsets)
    R.close(r.weights, weights, weights * bound, FULL)


@gpu
def test_route_strides_empty_and_infinite(F):
    x = torch.randn(70, 50, device="cuda")
    a, b = F.moe_route(x[:, 5:45], 4), F.moe_route(x[:, 5:45].contiguous(), 4)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    r = F.moe_route(x[:0], 4)
    assert r.experts.shape == (0, 4) and r.order.shape == (0,) and torch.equal(r.offsets, torch.zeros(51, dtype=torch.int32, device="cuda"))
    y = torch.zeros(1, 8, device="cuda")
    y[0, 5] = float("inf")
    r = F.moe_route(y, 2)
    assert r.experts.tolist() == [[5, 0]] and torch.isnan(r.weights[0, 0])


# ------------------------------------------------------------------------------------------ grouped products
def _groups(E, R_, seed, kind):
    """Row counts of E groups that sum to R_."""
    rng = np.random.default_rng(seed)
    if kind == "even":
        n = np.full(E, R_ // E)
        n[: R_ - n.sum()] += 1
    elif kind == "one":
        n = np.zeros(E, np.int64)
        n[E // 2] = R_
    else:
        n = rng.multinomial(R_, rng.dirichlet(np.full(E, 0.3)))
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int64)


def _grouped(F, E, R_, N, K, dtype, bias, act, kind, order=None, top_k=1, M=None):
    g = torch.Generator().manual_seed(E * 31 + R_ + N + K)
    M = R_ if M is None else M
    a, ad, sa = _codes(g, M, K)
    b, bd, sb = _codes(g, E * N, K)
    bd, sb = bd.unflatten(0, (E, N)), (sb / K ** 0.5).view(E, N)
    v = torch.randn(E, N, generator=g).to(dtype) if bias else None
    off = _groups(E, R_, R_, kind)
    rows = np.arange(R_) if order is None else np.asarray(order) // top_k
    want = np.zeros((R_, N // 2 if act == "swiglu" else N))
    err = np.zeros_like(want)
    bn = b.reshape(E, N, K)
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            r = rows[lo:hi]
            want[lo:hi], err[lo:hi] = R.product(a[r], sa.double().numpy()[r], bn[e], sb[e].double().numpy(), v[e].double().numpy() if bias else None, act)
    args = (ad, bd, sb.cuda(), torch.from_numpy(off).int().cuda(), v.cuda() if bias else None)
    kw = dict(a_scales=sa.cuda(), activation=act, dtype=dtype)
    if order is not None:
        kw.update(order=torch.as_tensor(np.asarray(order), dtype=torch.int32).cuda(), top_k=top_k)
    return args, kw, want, err


GROUPS = [(1, 40, 130, 70, "even"), (3, 0, 16, 32, "even"), (8, 8, 256, 300, "even"), (5, 33, 7, 100, "ragged"), (33, 64, 128, 2048, "ragged"),
          (64, 500, 384, 96, "ragged"), (12, 2000, 200, 1000, "ragged"), (7, 700, 1030, 64, "one"), (300, 900, 20, 33, "ragged"),
          (1024, 1500, 4, 16, "ragged"), (4, 1100, 2500, 256, "even"), (2, 1, 4096, 1024, "one"),
          (20, 6000, 1000, 700, "ragged"), (3, 2000, 3000, 130, "one"), (9, 9000, 1500, 900, "ragged"), (16, 4096, 2048, 640, "even"),
          (20, 3000, 1000, 1100, "ragged"), (3, 2000, 1502, 1030, "one"), (40, 9000, 1300, 100, "ragged")]


@gpu
@pytest.mark.parametrize("E,rows,N,K,kind", GROUPS)
@pytest.mark.parametrize("dtype,bias,act", [(HALF, True, "none"), (FULL, False, "none"), (HALF, False, "swiglu"), (FULL, True, "swiglu"), (FULL, True, "relu")])
def test_grouped_product(F, E, rows, N, K, kind, dtype, bias, act):
    args, kw, want, err = _grouped(F, E, rows, N + (N % 2 if act == "swiglu" else 0), K, dtype, bias, act, kind)
    R.close(F.matmul_int8_grouped(*args, **kw), want, err, dtype)
    assert F.device_error() == 0


@gpu
@pytest.mark.parametrize("T,E,k,N,K", [(1, 64, 8, 256, 512), (3, 8, 8, 130, 33), (70, 16, 2, 200, 100), (333, 12, 3, 100, 250), (700, 6, 4, 2500, 64), (40, 5, 1, 64, 16), (2000, 10, 3, 700, 1000), (1500, 16, 4, 256, 2048), (1200, 6, 2, 130, 4100)])
@pytest.mark.parametrize("dtype,act", [(HALF, "swiglu"), (FULL, "none")])
def test_grouped_product_of_gathered_tokens(F, T, E, k, N, K, dtype, act):
    order = np.random.default_rng(T).permutation(T * k)
    args, kw, want, err = _grouped(F, E, T * k, N, K, dtype, True, act, "ragged", order, k, T)
    y = F.matmul_int8_grouped(*args, **kw)
    R.close(y, want, err, dtype)
    # the same token many times, and rows in no order of tokens at all
    again = np.zeros(T * k, np.int64)
    args, kw, want, err = _grouped(F, E, T * k, N, K, dtype, True, act, "even", again, k, T)
    R.close(F.matmul_int8_grouped(*args, **kw), want, err, dtype)
    assert F.device_error() == 0


def _summed(want, err, slots, weights):
    """sum_j weights[t, j] row[slots[t, j]] and its bound: a float32 row each, k products and sums."""
    w = weights.astype(np.float64)[..., None]
    inside = ((slots >= 0) & (slots < len(want)))[..., None]
    at = np.clip(slots, 0, max(len(want) - 1, 0))
    rows, bounds = (np.where(inside, x[at] if len(x) else 0.0, 0.0) for x in (want, err))
    y = (w * rows).sum(1)
    size = (np.abs(w) * np.abs(rows)).sum(1)
    return y, (np.abs(w) * (bounds + R.EPS * np.abs(rows))).sum(1) + slots.shape[1] * R.EPS * size * 1.01 + 2.0 ** -140


@gpu
@pytest.mark.parametrize("T,E,k,N,K", [(1, 64, 8, 256, 512), (3, 8, 8, 130, 33), (70, 16, 2, 201, 100), (777, 12, 3, 1003, 1000), (40, 5, 1, 4, 16)])
@pytest.mark.parametrize("dtype,act", [(HALF, "none"), (FULL, "none"), (FULL, "swiglu")])
def test_grouped_product_summed_per_token(F, T, E, k, N, K, dtype, act):
    N += N % 2 if act == "swiglu" else 0
    args, kw, want, err = _grouped(F, E, T * k, N, K, dtype, True, act, "ragged")
    rng = np.random.default_rng(T + 1)
    slots = rng.permutation(T * k).reshape(T, k)
    slots[rng.random((T, k)) < 0.1] = -1
    if T > 10:
        slots[2, 0], slots[3, 0], slots[4, 0] = T * k, 1 << 30, slots[5, 0]  # beyond the rows: left out; the same row twice
    weights = rng.normal(size=(T, k)).astype(np.float32)
    y = F.matmul_int8_grouped(*args, **kw, slots=torch.from_numpy(slots).int().cuda(), weights=torch.from_numpy(weights).cuda())
    R.close(y, *_summed(want, err, slots, weights), dtype)
    assert F.device_error() == 0


@gpu
def test_grouped_rows_of_no_group(F):
    args, kw, want, err = _grouped(F, 4, 50, 60, 64, HALF, False, "none", "even")
    off = torch.tensor([5, 9, 9, 30, 41], dtype=torch.int32, device="cuda")
    args = args[:3] + (off,)
    y = F.matmul_int8_grouped(*args, **kw)
    assert (y[:5] == 0).all() and (y[41:] == 0).all()
    full = torch.full((50, 60), 3.0, dtype=HALF, device="cuda")
    F.matmul_int8_grouped(*args, **kw, out=full)
    assert torch.equal(full[5:41], y[5:41]) and (full[:5] == 3).all() and (full[41:] == 3).all()
    none = torch.zeros(5, dtype=torch.int32, device="cuda")
    assert (F.matmul_int8_grouped(*args[:3], none, **kw) == 0).all()
    slots = torch.tensor([[0, 10], [45, 49]], dtype=torch.int32, device="cuda")
    s = F.matmul_int8_grouped(*args, **kw, slots=slots, weights=torch.ones(2, 2, device="cuda"))
    assert torch.equal(s[0], y[10]) and (s[1] == 0).all()
    # no rows at all: sums of nothing
    s = F.matmul_int8_grouped(args[0][:0], *args[1:3], none, a_scales=kw["a_scales"][:0], slots=slots, weights=torch.ones(2, 2, device="cuda"))
    assert s.shape == (2, 60) and (s == 0).all()
    assert F.device_error() == 0


@gpu
def test_grouped_offsets_and_order_that_do_not_fit(F):
    args, kw, want, err = _grouped(F, 4, 50, 60, 64, FULL, False, "none", "even")
    good = F.matmul_int8_grouped(*args, **kw)
    first = args[3].tolist()
    for off, keep in (([0, first[1], first[2], first[3], 51], 3), ([-1] + first[1:], 0), ([0, first[1], first[2], 1 << 30, first[4]], 2),
                      ([0, first[2], first[1], first[3], first[4]], 1)):
        y = torch.full_like(good, 7.0)
        F.matmul_int8_grouped(*args[:3], torch.tensor(off, dtype=torch.int32, device="cuda"), **kw, out=y)
        assert F.device_error() == 0x701
        end = off[keep]  # the groups before the first bad offset; nothing behind them is written
        assert (y[end:] == 7).all() and torch.equal(y[:first[1]] if keep else y[:0], good[:first[1]] if keep else good[:0])
    many, kwm, want, err = _grouped(F, 300, 900, 20, 33, FULL, False, "none", "ragged")
    off = many[3].tolist()
    whole = F.matmul_int8_grouped(*many, **kwm)
    for bad in (5, 31, 32, 33, 100, 299):
        broken = many[3].clone()
        broken[bad + 1:] = -5
        y = torch.full_like(whole, 7.0)
        F.matmul_int8_grouped(*many[:3], broken, **kwm, out=y)
        assert F.device_error() == 0x701
        assert torch.equal(y[:off[bad]], whole[:off[bad]]) and (y[off[bad]:] == 7).all()
        y = F.matmul_int8_grouped(*many[:3], broken, **kwm)  # without out they are zero, in the sums too
        assert torch.equal(y[:off[bad]], whole[:off[bad]]) and (y[off[bad]:] == 0).all()
        slots = torch.randperm(900, device="cuda").int().view(450, 2)
        s = F.matmul_int8_grouped(*many[:3], broken, **kwm, slots=slots, weights=torch.ones(450, 2, device="cuda"))
        assert torch.equal(s, y[slots[:, 0].long()] + y[slots[:, 1].long()])
        assert F.device_error() == 0x701
    for off in ([-1] * 5, [51] * 5, [20, 10, 30, 40, 50], [7, 7, 7, 7, 51], [-1, 10, 20, 30, 50], [60, 10, 20, 30, 50]):
        y = F.matmul_int8_grouped(*args[:3], torch.tensor(off, dtype=torch.int32, device="cuda"), **kw)
        assert (y == 0).all() and F.device_error() == 0x701
    order = torch.arange(50, dtype=torch.int32, device="cuda")
    order[3], order[40] = -1, 50
    y = F.matmul_int8_grouped(*args, **kw, order=order)
    assert F.device_error() == 0x702
    keep = [i for i in range(50) if i not in (3, 40)]
    assert torch.equal(y[keep], good[keep]) and (y[3] == 0).all() and (y[40] == 0).all()


@gpu
def test_no_tokens_at_all(F):
    x, scores = torch.zeros(0, 64, dtype=HALF, device="cuda"), torch.zeros(0, 6, device="cuda")
    up, down = (F.int8_quantize(torch.ones(6, 64, 64, device="cuda")) for _ in range(2))
    r = F.moe_route(scores, 2)
    h = F.matmul_int8_grouped(x, *up, r.offsets, order=r.order, top_k=2)
    assert h.shape == (0, 64) and F.matmul_int8_grouped(h, *down, r.offsets, slots=r.slots, weights=r.weights).shape == (0, 64)
    assert F.matmul_int8(x, up[0][0], up[1][0]).shape == (0, 64)


@gpu
def test_c_calls_with_the_librarys_workspace(F, cuda_lib):
    """NULL workspaces: quantised rows, gathered rows, rows to be summed, a router's counts."""
    g = torch.Generator().manual_seed(8)
    E, T, k, N, K = 6, 300, 2, 130, 200
    x = torch.randn(T, K, generator=g, dtype=HALF).cuda()
    w, ws = F.int8_quantize(torch.randn(E, N, K, generator=g).cuda())
    scores = torch.randn(T, E, generator=g).cuda()
    r = F.moe_route(scores, k)
    own = [torch.empty_like(t) for t in r]
    p = _native.MoeRouteProblem_(_native.FLOAT32, 1, T, E, k, 0, scores.data_ptr(), *(t.data_ptr() for t in own))
    stream = torch.cuda.current_stream().cuda_stream
    assert cuda_lib.xrgpu_moe_route(ctypes.byref(p), None, 0, stream) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(own, r))
    y, s = torch.empty(T * k, N, dtype=HALF, device="cuda"), torch.empty(T, N, dtype=HALF, device="cuda")
    q = _native.Int8Problem_()
    q.dtype = q.a_dtype = _native.FLOAT16
    q.M, q.K, q.N, q.groups, q.rows, q.top_k = T, K, N, E, T * k, k
    q.a, q.b, q.b_scales, q.ldb, q.offsets, q.order, q.y = x.data_ptr(), w.data_ptr(), ws.data_ptr(), w.stride(1), r.offsets.data_ptr(), r.order.data_ptr(), y.data_ptr()
    assert cuda_lib.xrgpu_int8_forward(ctypes.byref(q), None, 0, stream) == 0
    assert torch.equal(y, F.matmul_int8_grouped(x, w, ws, r.offsets, order=r.order, top_k=k))
    q.slots, q.weights, q.tokens, q.y = r.slots.data_ptr(), r.weights.data_ptr(), T, s.data_ptr()
    assert cuda_lib.xrgpu_int8_forward(ctypes.byref(q), None, 0, stream) == 0
    assert torch.equal(s, F.matmul_int8_grouped(x, w, ws, r.offsets, order=r.order, top_k=k, slots=r.slots, weights=r.weights))
    assert F.device_error() == 0


@gpu
def test_sizes_beyond_32_bits(F):
    """More than 2^31 values of a result, of an operand's codes and of a row quantisation: the last rows are right."""
    g = torch.Generator(device="cuda").manual_seed(9)
    M, N, K = 66000, 33000, 32
    a = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    sa, sb = torch.full((M,), 2.0 ** -6, device="cuda"), torch.full((N,), 2.0 ** -6, device="cuda")
    y = F.matmul_int8(a, b, sb, a_scales=sa)
    for rows in (slice(0, 3), slice(M // 2, M // 2 + 3), slice(M - 3, M)):  # sums below 2^20, scaled by 2^-12: one rounding
        assert torch.equal(y[rows], (a[rows].double() @ b.double().t() * 2.0 ** -12).to(HALF))
    del a, b, y
    E, N, K = 5, 30000, 16400  # 2.46e9 codes; the last expert's begin at 1.97e9
    w = torch.zeros(E, N, K, dtype=torch.int8, device="cuda")
    w[3:, -300:] = torch.randint(-127, 128, (2, 300, K), generator=g, device="cuda", dtype=torch.int8)
    x = torch.randint(-9, 10, (20, K), generator=g, device="cuda", dtype=torch.int8)
    off = torch.tensor([0, 0, 3, 3, 9, 20], dtype=torch.int32, device="cuda")
    y = F.matmul_int8_grouped(x, w, torch.ones(E, N, device="cuda"), off, a_scales=torch.ones(20, device="cuda"), dtype=FULL)
    assert torch.equal(y[9:, -300:].double(), x[9:].double() @ w[4, -300:].double().t()) and (y[9:, :-300] == 0).all()
    assert torch.equal(y[3:9, -300:].double(), x[3:9].double() @ w[3, -300:].double().t()) and (y[:3] == 0).all()
    del w, y
    h = torch.zeros(70000, 31000, dtype=HALF, device="cuda")
    h[-2:] = torch.randn(2, 31000, generator=g, device="cuda", dtype=HALF)
    c, s = F.int8_quantize(h)
    codes, scales = R.quantize(h[-2:].cpu().double().numpy())
    assert np.array_equal(c[-2:].cpu().numpy(), codes) and np.array_equal(s[-2:].cpu().double().numpy(), scales) and not c[:-2].any()
    assert torch.equal(F.int8_dequantize(c, s, dtype=HALF)[-2:].cpu(), (torch.from_numpy(codes).float() * torch.from_numpy(scales).float()[:, None]).to(HALF))
    assert F.device_error() == 0


# ------------------------------------------------------------------------------------------ together
def _layer(F, x, scores, k, up, down, **kw):
    r = F.moe_route(scores, k)
    h = F.matmul_int8_grouped(x, *up, r.offsets, order=r.order, top_k=k, activation="swiglu")
    return r, h, F.matmul_int8_grouped(h, *down, r.offsets, slots=r.slots, weights=r.weights, **kw)


@gpu
@pytest.mark.parametrize("dtype", [HALF, FULL])
@pytest.mark.parametrize("T,E,k,hidden,inter", [(1, 16, 4, 256, 192), (9, 60, 6, 200, 72), (500, 8, 2, 384, 256)])
def test_mixture_of_experts(F, dtype, T, E, k, hidden, inter):
    """Router, both products and the sum, each step against the formula on what the step before gave."""
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, hidden, generator=g).to(dtype)
    scores = torch.randn(T, E, generator=g).to(dtype)
    up = F.int8_quantize((torch.randn(E, 2 * inter, hidden, generator=g) * hidden ** -0.5).cuda())
    down = F.int8_quantize((torch.randn(E, hidden, inter, generator=g) * inter ** -0.5).cuda())
    r, h, y = _layer(F, x.cuda(), scores.cuda(), k, up, down)
    experts, weights, order, slots, offsets, bound = R.route(scores.double().numpy(), k)
    assert np.array_equal(r.experts.cpu().numpy(), experts) and np.array_equal(r.slots.cpu().numpy(), slots)

    def products(codes, scales, rows, w, act):
        n = w[0].shape[1] // (2 if act == "swiglu" else 1)
        want, err = np.zeros((T * k, n)), np.zeros((T * k, n))
        for e in range(E):
            lo, hi = offsets[e], offsets[e + 1]
            if lo < hi:
                want[lo:hi], err[lo:hi] = R.product(codes[rows[lo:hi]], scales[rows[lo:hi]], w[0][e].cpu().numpy(), w[1][e].cpu().double().numpy(), None, act)
        return want, err

    want, err = products(*R.quantize(x.double().numpy()), order // k, up, "swiglu")
    R.close(h, want, err, dtype)
    want, err = products(*R.quantize(h.cpu().double().numpy()), np.arange(T * k), down, "none")
    R.close(y, *_summed(want, err, slots, r.weights.cpu().numpy()), dtype)
    # beside the experts as they were before quantisation: 8 bits on both sides of both products lose about a hundredth
    deq = [F.int8_dequantize(c, s).double().cpu() for c, s in (up, down)]
    plain = torch.zeros(T, hidden, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            z = deq[0][experts[t, j]] @ x[t].double()
            act = torch.from_numpy(R.swiglu(z[0::2].numpy(), z[1::2].numpy()))
            plain[t] += weights[t, j] * (deq[1][experts[t, j]] @ act)
    assert (y.cpu().double() - plain).norm() <= 0.05 * plain.norm()
    assert F.device_error() == 0


@gpu
def test_captured_layers_share_nothing(F):
    """Two captured layers, replayed in turn with new inputs, on a stream of their own, beside eager calls."""
    g = torch.Generator().manual_seed(5)
    E, k, hidden, inter = 12, 3, 320, 128
    up = F.int8_quantize(torch.randn(E, 2 * inter, hidden, generator=g).cuda())
    down = F.int8_quantize(torch.randn(E, hidden, inter, generator=g).cuda())
    made = []
    for T in (3, 150):
        x, scores = torch.randn(T, hidden, generator=g).cuda(), torch.randn(T, E, generator=g).cuda()
        _layer(F, x, scores, k, up, down)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _layer(F, x, scores, k, up, down)[2]
        made.append((graph, x, scores, y))
    side = torch.cuda.Stream()
    for turn in range(4):
        for graph, x, scores, y in made:
            x.copy_(torch.randn(x.shape, generator=g))
            scores.copy_(torch.randn(scores.shape, generator=g))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for graph, *_ in made:
                graph.replay()
        side.synchronize()
        for graph, x, scores, y in made:
            assert torch.equal(y, _layer(F, x, scores, k, up, down)[2])
    assert F.device_error() == 0


@gpu
def test_calls_on_two_streams(F):
    g = torch.Generator().manual_seed(6)
    w, s = F.int8_quantize(torch.randn(2048, 1024, generator=g).cuda())
    xs = [torch.randn(m, 1024, generator=g, dtype=HALF).cuda() for m in (1, 40, 300)]
    want = [F.matmul_int8(x, w, s) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(5):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(F.matmul_int8(x, w, s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))
