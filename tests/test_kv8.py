"""The paged 8-bit key/value cache: refusals on the CPU; append, read back and attention on the GPU against plain
64-bit restatements (serving_reference), and a decoder layer's run of the operators together."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as R
from xrgpu_b200 import _native

gpu = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def F(cuda_lib):
    from xrgpu_b200 import functional
    return functional


# ------------------------------------------------------------------------------------------ refusals (no GPU)
def _problem(**kw):
    p = _native.Kv8Problem_()
    p.dtype, p.cache_dtype, p.causal, p.scale = _native.FLOAT16, _native.INT8, 1, 0.125
    p.tokens, p.sequences, p.heads_q, p.heads_kv, p.head_dim, p.page, p.pages, p.max_pages = 2, 2, 4, 2, 64, 16, 4, 2
    for n in ("q", "k", "v", "o", "k_cache", "v_cache", "k_scale", "v_scale", "page_table", "kv_len"):
        setattr(p, n, 4096)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


BOTH = [
    (dict(dtype=_native.INT8), "T1"), (dict(cache_dtype=_native.UINT8), "cache codes"), (dict(head_dim=80), "head_dim"),
    (dict(page=24), "page"), (dict(page=256), "page"), (dict(tokens=-1), "geometry"), (dict(sequences=70000), "geometry"),
    (dict(heads_kv=0), "geometry"), (dict(max_pages=1 << 30), "geometry"), (dict(tokens=3), "multiple of sequences"),
    (dict(k_cache=4104), "aligned"), (dict(kv_len=None), "null"), (dict(page_table=None), "null"), (dict(v_scale=None), "null"),
]


@pytest.mark.parametrize("change,message", BOTH + [(dict(k=None), "null"), (dict(k_stride=127), "stride"), (dict(v_stride=1), "stride")])
def test_append_refusals(cuda_lib, change, message):
    for fn in (cuda_lib.xrgpu_kv8_append, cuda_lib.xrgpu_kv8_read):
        assert fn(ctypes.byref(_problem(**change)), None) == _native.INVALID_ARGUMENT
        assert message in cuda_lib.xrgpu_last_error().decode()


@pytest.mark.parametrize("change,message", BOTH + [
    (dict(heads_q=3), "heads_q"), (dict(heads_q=0), "heads_q"), (dict(window=-1), "window"), (dict(window=4, causal=0), "window"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(o=None), "null"),
    (dict(q_stride=255), "stride"), (dict(o_stride=255), "stride"), (dict(tokens=1 << 30, sequences=1), "geometry")])
def test_attention_refusals(cuda_lib, change, message):
    assert cuda_lib.xrgpu_kv8_attention(ctypes.byref(_problem(**change)), None, 0, None) == _native.INVALID_ARGUMENT
    assert message in cuda_lib.xrgpu_last_error().decode()


def test_empty_calls_need_no_gpu(cuda_lib):
    for change in (dict(tokens=0), dict(sequences=0, tokens=0)):
        assert cuda_lib.xrgpu_kv8_attention(ctypes.byref(_problem(**change)), None, 0, None) == 0
        need = ctypes.c_uint64(7)
        assert cuda_lib.xrgpu_kv8_attention_workspace_size(ctypes.byref(_problem(**change)), ctypes.byref(need)) == 0
        assert need.value == 0


def test_python_refusals(F):
    c = R.Cache([20, 3], heads=2, D=64, page=16, code=INT8)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        F.attention_kv8(q, c.k, c.v, c.ks, c.vs, c.table, None, c.lens)
    with pytest.raises(ValueError, match="int8 or float8"):
        F.attention_kv8(q, c.k.float(), c.v, c.ks, c.vs, c.table, None, c.lens)
    with pytest.raises(ValueError, match="page, head_dim"):
        F.attention_kv8(q, c.k[0], c.v, c.ks, c.vs, c.table, None, c.lens)


# ------------------------------------------------------------------------------------------ append, read back
def _cu(new):
    return torch.tensor([0] + list(new), dtype=torch.int32).cumsum(0).to(torch.int32)


APPEND = [
    # past, new per sequence
    ([0], [1]), ([15], [1]), ([16], [1]), ([5, 0, 33], [1, 1, 1]), ([0, 7], [40, 1]), ([3, 16, 0, 100], [0, 17, 129, 2]),
    ([31], [32]), ([250], [300]),
]


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("page,D", [(16, 64), (64, 128), (128, 64), (32, 128)])
@pytest.mark.parametrize("past,new", APPEND)
def test_append_is_exact(F, code, dtype, page, D, past, new):
    c = R.Cache([a + b for a, b in zip(past, new)], heads=3, D=D, page=page, code=code, seed=page + D)
    c.poison_tails()
    T = sum(new)
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(T, 3, D, generator=g).to(dtype) * torch.where(torch.rand(T, 3, 1, generator=g) < 0.3, 6.0, 0.5).to(dtype) for _ in range(2))
    cu = _cu(new)
    dev = c.cuda()
    F.kv8_append(k.cuda(), v.cuda(), *dev, cu.cuda(), c.lens.cuda())
    R.append(c, k, v, cu)
    for got, want in zip(dev[:4], (c.k, c.v, c.ks, c.vs)):
        as_bytes = lambda t: t.cpu().contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int32)  # noqa: E731
        # codes may differ in the sign of zero only (e4m3)
        same = (as_bytes(got) == as_bytes(want)) | ((as_bytes(got) & 0x7F) + (as_bytes(want) & 0x7F) == 0 if code == E4M3 and got.element_size() == 1 else False)
        both_nan = torch.isnan(got.cpu()) & torch.isnan(want) if got.dtype == torch.float32 else torch.tensor(False)
        assert bool((same | both_nan).all())
    # what the cache holds for the new tokens, rounded once to the rows' type
    rk, rv = F.kv8_read(*dev, cu.cuda(), c.lens.cuda(), rows=T, dtype=dtype)
    for got, which in ((rk, 0), (rv, 1)):
        want = np.concatenate([c.tokens(b)[which][past[b]:] for b in range(len(new))])
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(dtype))


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
def test_append_borders_round_to_even(F, code):
    """Quotients that lie on and next to the borders between codes, with scales that are no powers of two."""
    D, L = 64, R.LIMIT[code]
    x = torch.zeros(16, 1, D)
    rng = np.random.default_rng(3)
    for t in range(16):
        a = np.float32(rng.uniform(1, 9))
        s = np.float32(a / np.float32(L))
        q = rng.integers(-126, 126, D) + 0.5 if code == INT8 else np.ldexp(rng.integers(8, 16, D) + 0.5, rng.integers(-5, 5, D))
        v = (np.abs(q) * np.float64(s)).astype(np.float32)  # the float32 numbers next to the borders
        v = np.nextafter(v, np.where(rng.random(D) < 0.5, np.float32(0), np.float32(1e9))) if t % 2 else v
        x[t, 0] = torch.from_numpy(v.astype(np.float32))
        x[t, 0, 0] = float(a)
    x = x.clamp(max=float(x[:, 0, 0].max()))
    for n in range(16):  # a page of its own for each, so that each has its own scale
        c = R.Cache([1], heads=1, D=D, page=16, code=code, seed=n)
        dev = c.cuda()
        row = x[n:n + 1]
        F.kv8_append(row.cuda(), row.cuda(), *dev, _cu([1]).cuda(), c.lens.cuda())
        R.append(c, row, row, _cu([1]))
        assert torch.equal(dev[0].cpu().float(), c.k.float()) and torch.equal(dev[2].cpu(), c.ks)


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("size", [2.0 ** -149, 2.0 ** -142, 2.0 ** -130, 1e-30, 2.0 ** -58, 2.0 ** -52, 1e25, 3e38])
def test_append_extreme_magnitudes(F, code, size):
    """Scales that are subnormal, or whose reciprocals leave the normal range; older codes under them."""
    g = torch.Generator().manual_seed(7)
    for past in (0, 9):
        c = R.Cache([past + 40], heads=2, D=64, page=32, code=code)
        if past:
            c.ks[c.table[0, 0]] = float(np.float32(size * 2.0 ** -9))
            c.vs[c.table[0, 0]] = float(np.float32(size * 2.0 ** -7))
        dev = c.cuda()
        k, v = ((torch.rand(40, 2, 64, generator=g, dtype=torch.float64) * 2 - 1) * size * f for f in (1.0, 250.0 if size < 1e30 else 0.3))
        k, v = k.float(), v.float()
        F.kv8_append(k.cuda(), v.cuda(), *dev, _cu([40]).cuda(), c.lens.cuda())
        R.append(c, k, v, _cu([40]))
        for i in (0, 1):
            assert torch.equal(dev[i + 2].cpu(), (c.ks, c.vs)[i])
            assert torch.equal(dev[i].cpu().float(), (c.k, c.v)[i].float())


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
def test_append_token_by_token_rescales(F, code):
    """Growing values rescale a page again and again; the state stays the definition's."""
    c = R.Cache([0], heads=2, D=64, page=32, code=code, max_extra=3)
    c.table[0, :3] = torch.tensor([2, 0, 1])
    c = R.Cache([70], heads=2, D=64, page=32, code=code)
    dev = c.cuda()
    for i in range(70):
        c.lens[0] = i + 1
        k = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(i)) * (1.0 + 0.2 * i)
        v = k.flip(-1) * (0.1 if i % 3 else 0.0)
        F.kv8_append(k.cuda(), v.cuda(), *dev, _cu([1]).cuda(), c.lens.cuda())
        R.append(c, k, v, _cu([1]))
    ids = c.table[0, :3].long()
    for got, want in zip(dev[:2], (c.k, c.v)):
        w = want[ids].float().transpose(1, 2).reshape(-1, 2, 64)[:70]
        assert torch.equal(got.cpu()[ids].float().transpose(1, 2).reshape(-1, 2, 64)[:70], w)
    assert torch.equal(dev[2].cpu()[ids], c.ks[ids]) and torch.equal(dev[3].cpu()[ids], c.vs[ids])


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
def test_append_non_finite_poisons_its_block_only(F, code):
    c = R.Cache([20, 18], heads=2, D=64, page=16, code=code)
    dev = c.cuda()
    k = torch.randn(6, 2, 64)
    v = torch.randn(6, 2, 64)
    k[1, 0, 3], v[5, 1, 60] = float("nan"), float("-inf")
    cu = _cu([4, 2])
    F.kv8_append(k.cuda(), v.cuda(), *dev, cu.cuda(), c.lens.cuda())
    R.append(c, k, v, cu)
    for got, want in zip(dev[2:4], (c.ks, c.vs)):
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert int(torch.isnan(want).sum()) == 1


@gpu
def test_append_refuses_bad_pages_and_lengths(F):
    """Bad page ids, lengths past the table, more rows than tokens: recorded, nothing written for them."""
    F.device_error(0)
    for change, code in ((lambda c, cu: c.table.__setitem__((0, 1), 99), 0x501), (lambda c, cu: c.table.__setitem__((0, 1), -1), 0x501),
                         (lambda c, cu: c.lens.__setitem__(0, 3), 0x502), (lambda c, cu: c.lens.__setitem__(0, 10 ** 6), 0x502),
                         (lambda c, cu: cu.__setitem__(1, -5), 0x502), (lambda c, cu: c.lens.__setitem__(0, -1), 0x502)):
        c = R.Cache([20, 18], heads=1, D=64, page=16, code=INT8)
        cu = _cu([4, 2])
        change(c, cu)
        dev = c.cuda()
        k = torch.randn(6, 1, 64).cuda()
        F.kv8_append(k, k, *dev, cu.cuda(), c.lens.cuda())
        assert F.device_error(0) == code
        first = c.table[1, 1].item()  # of the pages, only the second sequence's may have changed
        keep = [i for i in range(c.k.shape[0]) if i != first]
        assert torch.equal(dev[0].cpu()[keep], c.k[keep]) and torch.equal(dev[2].cpu()[keep], c.ks[keep])
        F.attention_kv8(torch.randn(6, 1, 64).cuda(), *dev, cu.cuda(), c.lens.cuda())
        F.kv8_read(*dev, cu.cuda(), c.lens.cuda(), rows=6)
        F.device_error(0)
    assert F.device_error(0) == 0


@gpu
def test_append_strided_rows_and_rows_behind_the_last_sequence(F):
    c = R.Cache([20, 5], heads=2, D=64, page=16, code=INT8)
    fused = torch.randn(9, 8 * 64).half()
    k, v = fused[:, 128:256].unflatten(1, (2, 64)), fused[:, 256:384].unflatten(1, (2, 64))
    cu = _cu([4, 3])  # two padding rows
    dev, d2 = c.cuda(), c.cuda()
    fd = fused.cuda()
    F.kv8_append(fd[:, 128:256].unflatten(1, (2, 64)), fd[:, 256:384].unflatten(1, (2, 64)), *dev, cu.cuda(), c.lens.cuda())
    R.append(c, k.contiguous(), v.contiguous(), cu)
    assert torch.equal(dev[0].cpu(), c.k) and torch.equal(dev[1].cpu(), c.v)
    odd = torch.zeros(9, 130 + 1, dtype=torch.float16, device="cuda")[:, 1:129].unflatten(1, (2, 64))  # no 16-byte rows
    odd.copy_(fd[:, 128:256].unflatten(1, (2, 64)))
    F.kv8_append(odd, fd[:, 256:384].unflatten(1, (2, 64)), *d2, cu.cuda(), c.lens.cuda())
    assert torch.equal(d2[0].cpu(), c.k) and torch.equal(d2[1].cpu(), c.v)
    rk, _ = F.kv8_read(*dev, cu.cuda(), c.lens.cuda(), rows=9)
    assert bool((rk[7:] == 0).all())


# ------------------------------------------------------------------------------------------ attention
def _check(F, c, new, hq, dtype, *, pad=0, q=None, uniform=False, **kw):
    cu = _cu(new)
    T = sum(new) + pad
    if q is None:
        q = torch.randn(T, hq, c.D, generator=torch.Generator().manual_seed(T + hq)).to(dtype)
    want, tol = R.attention(c, q, cu, **kw)
    got = F.attention_kv8(q.cuda(), *c.cuda(), None if uniform else cu.cuda(), c.lens.cuda(), **kw)
    torch.cuda.synchronize()
    assert F.device_error(0) == 0
    g = got.cpu().double().numpy()[:sum(new)]
    assert np.isfinite(g).all()
    off = np.abs(g - want[:sum(new)]) - tol[:sum(new)]
    assert (off <= 0).all(), float(off.max())
    return got


LENS = [
    # lengths, new rows
    ([1], [1]), ([17], [1]), ([64], [1]), ([300, 1, 65], [1, 1, 1]), ([2000], [1]), ([129, 40, 16], [5, 2, 9]), ([200], [200]),
    ([77, 530], [33, 130]), ([40, 0, 90], [40, 0, 3]),
]


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,page,hq,hkv", [(128, 64, 8, 2), (64, 16, 5, 1), (128, 32, 12, 1), (64, 128, 3, 3)])
@pytest.mark.parametrize("lens,new", LENS)
def test_attention(F, code, dtype, D, page, hq, hkv, lens, new):
    c = R.Cache(lens, heads=hkv, D=D, page=page, code=code, seed=D + hq)
    c.poison_tails()
    _check(F, c, new, hq, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("window", [1, 7, 16, 100, 5000])
@pytest.mark.parametrize("lens,new", [([150], [1]), ([333, 20], [50, 20]), ([600], [140])])
def test_attention_window(F, dtype, window, lens, new):
    c = R.Cache(lens, heads=2, D=128, page=32, code=INT8)
    c.poison_tails()
    _check(F, c, new, 8, dtype, window=window)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("lens,new", [([40], [3]), ([100, 7], [20, 7]), ([5], [9]), ([290], [150])])
def test_attention_without_causal_mask(F, dtype, lens, new):
    c = R.Cache(lens, heads=2, D=64, page=16, code=E4M3)
    c.poison_tails()
    _check(F, c, new, 4, dtype, causal=False, scale=0.05)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_that_see_nothing_are_zero(F, dtype):
    """Empty sequences, and more rows than tokens: their first rows see nothing."""
    c = R.Cache([0, 3, 0], heads=2, D=64, page=16, code=INT8)
    got = _check(F, c, [2, 5, 1], 4, dtype)
    assert bool((got[:4] == 0).all()) and bool((got[7:] == 0).all()) and bool((got[4:7] != 0).any())
    _check(F, R.Cache([0, 50], heads=1, D=128, page=32, code=E4M3), [150, 180], 2, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("new", [[3, 2], [70, 130]])
def test_rows_behind_the_last_sequence_are_left(F, dtype, new):
    c = R.Cache([150, 200], heads=2, D=128, page=64, code=INT8)
    q = torch.randn(sum(new) + 9, 8, 128, device="cuda", dtype=dtype)
    q[sum(new):] = float("nan")
    out = torch.full_like(q, 3.0)
    cu = _cu(new).cuda()
    F.attention_kv8(q, *c.cuda(), cu, c.lens.cuda(), out=out)
    assert bool((out[sum(new):] == 3.0).all()) and bool(torch.isfinite(out[:sum(new)]).all())
    fresh = F.attention_kv8(q, *c.cuda(), cu, c.lens.cuda())
    assert torch.equal(fresh[:sum(new)], out[:sum(new)]) and bool((fresh[sum(new):] == 0).all())


# Calls with enough rows for the prompt kernel: the key/value heads that it takes.
def _heads(new, G, D):
    B = len(new)
    rows = -(-sum(new) // B) * G
    heads = 1
    while B * heads * rows * D < 6500 * 128 * -(-(B * heads * -(-rows // 256)) // 148):
        heads += 1
    assert rows > 64
    return heads


PROMPTS = [
    ([200], [200], {}), ([77, 530], [33, 130], {}), ([700, 30, 1], [260, 30, 1], {}), ([40, 0, 290], [40, 0, 150], {}),
    ([333, 20], [150, 20], {"window": 100}), ([300], [140], {"window": 7}), ([333, 300], [100, 260], {"window": 1}),
    ([200, 7], [120, 7], {"causal": False, "scale": 0.05}), ([90], [150], {"causal": False}), ([290], [150], {"scale": -0.1}),
    ([0, 50], [150, 180], {}),  # more rows than tokens
]


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("D,page,G", [(128, 64, 4), (64, 16, 5), (128, 32, 2), (64, 128, 3)])
@pytest.mark.parametrize("lens,new,kw", PROMPTS)
def test_prompts(F, code, D, page, G, lens, new, kw):
    heads = _heads(new, G, D)
    c = R.Cache(lens, heads=heads, D=D, page=page, code=code, seed=D + G)
    c.poison_tails()
    _check(F, c, new, G * heads, torch.float16, **kw)


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
def test_prompts_extreme_scores_and_scales(F, code):
    new = [260, 150]
    heads = _heads(new, 4, 64)
    c = R.Cache([500, 300], heads=heads, D=64, page=16, code=code)
    c.vs *= torch.exp2(torch.randint(-10, 10, c.vs.shape, generator=torch.Generator().manual_seed(1)).float())
    c.ks[::3] *= 40.0
    _check(F, c, new, 4 * heads, torch.float16)
    c.ks.zero_()
    c.vs[::2] = 0.0
    _check(F, c, new, 4 * heads, torch.float16)


@gpu
def test_prompts_leave_rows_and_repeat(F):
    """Strided queries and results, rows behind the last sequence, no cu_seqlens, the same bits on every call."""
    new = [130, 130]
    heads = _heads(new, 2, 128)
    c = R.Cache([150, 200], heads=heads, D=128, page=64, code=INT8)
    dev, hq, n = c.cuda(), 2 * heads, 260
    wide = torch.randn(n + 9, hq * 128 + 24, device="cuda", dtype=torch.float16)
    wide[n:] = float("nan")
    q = wide[:, 3:3 + hq * 128].unflatten(1, (hq, 128))
    out = torch.full((n + 9, hq * 128 + 40), 3.0, device="cuda", dtype=torch.float16)[:, 5:5 + hq * 128].unflatten(1, (hq, 128))
    F.attention_kv8(q, *dev, _cu(new).cuda(), c.lens.cuda(), out=out)
    assert bool((out[n:] == 3.0).all()) and bool(torch.isfinite(out[:n]).all())
    fresh = F.attention_kv8(q, *dev, _cu(new).cuda(), c.lens.cuda())
    assert torch.equal(fresh[:n], out[:n]) and bool((fresh[n:] == 0).all())
    assert torch.equal(F.attention_kv8(q[:n].contiguous(), *dev, None, c.lens.cuda()), out[:n])
    _check(F, c, new, hq, torch.float16, q=q[:n].cpu().contiguous(), uniform=True)


@gpu
def test_prompts_nan_blocks_reach_their_readers_only(F):
    new = [1, 170]
    heads = _heads(new, 2, 64)
    c = R.Cache([100, 180], heads=heads, D=64, page=16, code=INT8)
    q = torch.randn(sum(new), 2 * heads, 64, device="cuda", dtype=torch.float16)
    for side, keep in (("vs", 1.0), ("ks", 0.02)):
        for b, rows in ((0, slice(0, 1)), (1, slice(1 + 22, 171))):  # page 2 of the prompt: its rows from position 32 on
            at = getattr(c, side)
            at[c.table[b, 2], 1] = float("nan")
            o = F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda())
            nan = torch.isnan(o)
            want = torch.zeros_like(nan)
            want[rows, 2:4] = True
            assert torch.equal(nan, want)
            at[c.table[b, 2], 1] = keep


@gpu
def test_prompts_bad_pages_are_skipped(F):
    new = [150, 150]
    heads = _heads(new, 2, 64)
    c = R.Cache([170, 170], heads=heads, D=64, page=16, code=INT8)
    q = torch.randn(300, 2 * heads, 64, device="cuda", dtype=torch.float16)
    whole = F.attention_kv8(q, *c.cuda(), None, c.lens.cuda())
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        c.table[0, 1] = bad
        o = F.attention_kv8(q, *c.cuda(), None, c.lens.cuda())
        assert F.device_error(0) == 0x501
        assert bool(torch.isfinite(o).all()) and torch.equal(o[150:], whole[150:])
    for bad in (-3, 10 ** 6):
        c.lens[0] = bad
        o = F.attention_kv8(q, *c.cuda(), None, c.lens.cuda())
        assert F.device_error(0) == 0x502 and torch.equal(o[150:], whole[150:]) and bool((o[:150] == 0).all())


@gpu
def test_rows_without_sequences_are_zero(F):
    c = R.Cache([3], heads=2, D=64, page=16, code=INT8).cuda()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table, cu = none.view(0, 4), torch.zeros(1, dtype=torch.int32, device="cuda")
    junk = [torch.full((5, 4, 64), float("nan"), device="cuda") for _ in range(3)]  # what the allocator hands out next
    del junk
    q = torch.randn(5, 4, 64, device="cuda")
    assert not F.attention_kv8(q, *c[:4], table, cu, none).any()
    k, v = F.kv8_read(*c[:4], table, cu, none, rows=5, dtype=torch.float32)
    assert not k.any() and not v.any()
    out = torch.ones_like(q)
    F.attention_kv8(q, *c[:4], table, cu, none, out=out)
    assert bool((out == 1).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_extreme_scores_and_scales(F, dtype):
    """One token that takes all the weight, scores in the thousands, and value blocks of scales 2^20 apart."""
    c = R.Cache([500, 300], heads=1, D=64, page=16, code=INT8)
    c.vs *= torch.exp2(torch.randint(-10, 10, c.vs.shape).float())
    c.ks[::3] *= 40.0
    _check(F, c, [1, 2], 4, dtype)
    c.ks.zero_()
    c.vs[::2] = 0.0
    _check(F, c, [1, 2], 4, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("new", [[1, 1], [1, 150]])
def test_nan_blocks_reach_their_readers_only(F, dtype, new):
    c = R.Cache([100, 160], heads=2, D=64, page=16, code=INT8)
    c.vs[c.table[0, 2], 1] = float("nan")
    q = torch.randn(sum(new), 4, 64, device="cuda", dtype=dtype)
    o = F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda())
    assert bool(torch.isnan(o[0, 2:]).all()) and bool(torch.isfinite(o[0, :2]).all()) and bool(torch.isfinite(o[1:]).all())
    c.vs[c.table[0, 2], 1] = 1.0
    c.ks[c.table[0, 2], 0] = float("nan")
    o = F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda())
    assert bool(torch.isnan(o[0, :2]).all()) and bool(torch.isfinite(o[0, 2:]).all()) and bool(torch.isfinite(o[1:]).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_nan_page_at_the_edge_of_what_rows_see(F, dtype, page):
    """A page that only some rows of a tile see (behind the causal edge, or out of the window) reaches those only."""
    n, lens = 6, 3 * page + 2  # the last two rows are the first tokens of the last page
    for window in (0, page):
        for side in ("ks", "vs"):
            c = R.Cache([lens], heads=1, D=64, page=page, code=INT8)
            bad = 3 if window == 0 else 2
            getattr(c, side)[c.table[0, bad], 0] = float("nan")
            if window:
                c.ks[c.table[0, 3], 0] = 0.02
            q = torch.randn(n, 4, 64, device="cuda", dtype=dtype)
            o = F.attention_kv8(q, *c.cuda(), None, c.lens.cuda(), window=window)
            pos = torch.arange(lens - n, lens)
            lo = (pos - window + 1).clamp(min=0) if window else torch.zeros_like(pos)
            sees = (pos >= bad * page) & (lo < (bad + 1) * page)
            assert torch.equal(torch.isnan(o).all(-1).all(-1).cpu(), sees) and torch.equal(torch.isnan(o).any(-1).any(-1).cpu(), sees)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strides_uniform_and_repeat(F, dtype):
    """Queries inside a fused projection, an output with padding, no cu_seqlens; the same bits on every call."""
    c = R.Cache([90, 33], heads=2, D=64, page=16, code=INT8)
    fused = torch.randn(6, 1000, device="cuda", dtype=dtype)
    q = fused[:, 3:3 + 256].unflatten(1, (4, 64))
    out = torch.zeros(6, 300, device="cuda", dtype=dtype)[:, :256].unflatten(1, (4, 64))
    F.attention_kv8(q, *c.cuda(), None, c.lens.cuda(), out=out)
    want = F.attention_kv8(q.contiguous(), *c.cuda(), _cu([3, 3]).cuda(), c.lens.cuda())
    assert torch.equal(out, want)
    _check(F, c, [3, 3], 4, dtype, q=q.cpu().contiguous(), uniform=True)
    for _ in range(3):
        assert torch.equal(F.attention_kv8(q, *c.cuda(), None, c.lens.cuda()), want)


@gpu
def test_attention_bad_pages_are_skipped(F):
    """A bad page id is recorded and its tokens are left out; a bad length gives its rows zeros."""
    c = R.Cache([40, 40], heads=1, D=64, page=16, code=INT8)
    q = torch.randn(2, 2, 64, dtype=torch.float16)
    whole = F.attention_kv8(q.cuda(), *c.cuda(), None, c.lens.cuda())
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        c.table[0, 1] = bad
        o = F.attention_kv8(q.cuda(), *c.cuda(), None, c.lens.cuda())
        assert F.device_error(0) == 0x501
        assert bool(torch.isfinite(o).all()) and torch.equal(o[1], whole[1])
    for bad in (-3, 10 ** 6):
        c.lens[0] = bad
        o = F.attention_kv8(q.cuda(), *c.cuda(), None, c.lens.cuda())
        assert F.device_error(0) == 0x502 and torch.equal(o[1], whole[1]) and bool((o[0] == 0).all())


@gpu
def test_offsets_past_32_bits(F):
    """Pages whose codes lie more than 2^32 bytes into the cache."""
    P, H, page, D = 36000, 8, 128, 128  # 4.7 GB a side
    k = torch.zeros(P, H, page, D, dtype=torch.int8, device="cuda")
    v = torch.zeros(P, H, page, D, dtype=torch.int8, device="cuda")
    ks, vs = torch.ones(P, H, device="cuda"), torch.ones(P, H, device="cuda")
    table = torch.tensor([[P - 1, 5, P - 2]], dtype=torch.int32, device="cuda")
    kn, vn = (torch.randn(300, H, D, device="cuda", dtype=torch.float16) for _ in range(2))
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    F.kv8_append(kn, vn, k, v, ks, vs, table, None, lens)
    small = [t[[P - 1, 5, P - 2]].contiguous() for t in (k, v, ks, vs)]
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    for rows in (1, 200):
        q = torch.randn(rows, 16, D, device="cuda", dtype=torch.float16)
        o = F.attention_kv8(q, k, v, ks, vs, table, None, lens)
        assert torch.equal(o, F.attention_kv8(q, *small, near, None, lens)) and bool((o != 0).any())
    assert F.device_error(0) == 0


# ------------------------------------------------------------------------------------------ together
@gpu
def test_graphs_share_nothing(F):
    """A decode step (append, then attention) captured twice for two batches, replayed interleaved with new tokens."""
    steps = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for seed, lens in ((1, [700, 40]), (2, [1300, 5])):
        c = R.Cache([n + 40 for n in lens], heads=2, D=64, page=16, code=INT8, seed=seed)
        dev, n = c.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        q, k, v = (torch.randn(2, h, 64, device="cuda", dtype=torch.float16) for h in (8, 2, 2))

        def step(dev=dev, n=n, q=q, k=k, v=v):
            F.kv8_append(k, v, *dev, None, n)
            return F.attention_kv8(q, *dev, None, n)

        with torch.cuda.stream(side):
            step()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                o = step()
        steps.append((c, dev, n, q, k, v, g, o, step))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, dev, n, q, k, v, g, o, step in steps:
            n += 1
            for t in (q, k, v):
                t.copy_(torch.randn_like(t))
        torch.cuda.synchronize()
        for s in steps:
            s[6].replay()
        torch.cuda.synchronize()
        for c, dev, n, q, k, v, g, o, step in steps:
            got = o.clone()
            assert torch.equal(got, step())  # appending the same tokens again changes nothing
    assert F.device_error(0) == 0


@gpu
def test_decoder_layer_prompt_then_tokens(F):
    """qkv projection -> append -> attention -> output projection in 4-bit floating point, a prompt and then tokens
    one by one, against the same in float64 from the values that the cache holds."""
    hidden, hq, hkv, D, page = 512, 8, 2, 64, 16
    g = torch.Generator().manual_seed(5)
    kb = hidden // 32
    w = {n: (torch.randint(0, 256, (rows, kb, 16), generator=g, dtype=torch.uint8).cuda(), (torch.rand(rows, kb, generator=g) * 0.01).half().cuda())
         for n, rows in (("q", hq * D), ("k", hkv * D), ("v", hkv * D))}
    norm = torch.ones(hidden, dtype=torch.float16, device="cuda")
    oc, osc = F.mxfp4_quantize(torch.randn(hidden, hq * D, generator=g).cuda() * 0.05)
    o_values = F.mxfp4_dequantize(oc, osc).double().cpu().numpy()
    c = R.Cache([60, 45], heads=hkv, D=D, page=page, code=INT8)
    dev = c.cuda()
    lens = [0, 0]
    for new in ([37, 20], [1, 1], [1, 1], [3, 0]):
        lens = [a + b for a, b in zip(lens, new)]
        n, cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), _cu(new).cuda()
        x = torch.randn(sum(new), hidden, generator=g).half().cuda()
        q, k, v = F.matmul_nbits_qkv(x, norm, *w["q"], *w["k"], *w["v"])
        F.kv8_append(k.view(-1, hkv, D), v.view(-1, hkv, D), *dev, cu, n)
        o = F.attention_kv8(q.view(-1, hq, D), *dev, cu, n)
        y = F.matmul_mxfp4(o.view(-1, hq * D), oc, osc, dtype=torch.float32)
        held = R.Cache.__new__(R.Cache)
        held.__dict__.update(c.__dict__)
        held.k, held.v, held.ks, held.vs = (t.cpu() for t in dev[:4])
        held.lens = n.cpu()
        want, tol = R.attention(held, q.cpu().view(-1, hq, D), cu.cpu())
        assert (np.abs(o.cpu().double().numpy() - want) <= tol).all()
        _, _, xo = R.mx_quantize(o.cpu().double().numpy().reshape(sum(new), -1))
        yy = xo @ o_values.T
        assert (np.abs(y.cpu().double().numpy() - yy) <= (hq * D / 32 + 24) * 2.0 ** -23 * (np.abs(xo) @ np.abs(o_values).T)).all()
    assert F.device_error(0) == 0


# ------------------------------------------------------------------------------------------ limits of what rows see
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 64])
@pytest.mark.parametrize("lens,new", [([5], [9]), ([5, 60], [9, 3]), ([50], [180]), ([0, 50], [150, 180])])
def test_the_largest_windows_see_everything(F, dtype, window, lens, new):
    """Windows of as many tokens as a sequence holds are none, also where the first rows lie before the first token."""
    G, D = 4, 64
    heads = _heads(new, G, D) if max(new) > 100 else 2  # the long ones reach the prompt kernel with float16 rows
    c = R.Cache(lens, heads=heads, D=D, page=16, code=INT8)
    c.poison_tails()
    got = _check(F, c, new, G * heads, dtype, window=window)
    assert bool((got != 0).any())
    q = torch.randn(sum(new), G * heads, D, generator=torch.Generator().manual_seed(sum(new) + G * heads)).to(dtype)
    assert torch.equal(got, F.attention_kv8(q.cuda(), *c.cuda(), _cu(new).cuda(), c.lens.cuda(), window=0))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("lens,new", [([200, 90], [1, 3]), ([150 + 7 * i for i in range(40)], [1] * 40), ([333, 300], [150, 140])])
def test_pages_in_front_of_the_window_may_be_gone(F, dtype, page, lens, new):
    """Pages whose tokens no row sees any more are released (-1) as a window moves on: nothing is looked up there, nothing
    recorded, and the results are those with the pages still in place."""
    G = 4
    heads = _heads(new, G, 64) if max(new) > 100 else 2
    for window in (1, 40, 45, 64):
        c = R.Cache(lens, heads=heads, D=64, page=page, code=INT8)
        q = torch.randn(sum(new), G * heads, 64, dtype=dtype, device="cuda")
        want = F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda(), window=window)
        assert F.device_error(0) == 0
        gone = 0
        for b, (n, m) in enumerate(zip(lens, new)):
            first = max(0, n - m - window + 1)
            c.table[b, :first // page] = -1
            gone += first // page
        assert gone > 0
        got = F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda(), window=window)
        assert F.device_error(0) == 0
        assert torch.equal(got, want)
        # a page that a row does see is still missed
        c.table[0, (lens[0] - 1) // page] = -1
        F.attention_kv8(q, *c.cuda(), _cu(new).cuda(), c.lens.cuda(), window=window)
        assert F.device_error(0) == 0x501


# ------------------------------------------------------------------------------------------ float32 rows
def _float32_bound(k, v, q, scale):
    """(o, tolerance) float64 of one float32 row over keys and values [n, D]: float32 sums over D products in a score, each
    counted once in the values' sum and once in the normaliser, as are an exponential's 2^-21 and the weight's
    rounding. A weight is a pair of float16 numbers, the second 2^11 times the rest, of 2^7 to 2^15 for the largest: 2^-24 of
    itself, and steps of 2^-25 2^-11 2^-7 = 2^-43 of the largest where the second number is a subnormal. A
    query is a pair of float16 numbers below 2^15: 2^-24 of itself (one product's rounding), and steps of 2^-25 2^-14 = 2^-39
    of the row's largest. n tokens summed in float32 in steps of 32 by at least six warps."""
    n, D = k.shape
    x = k @ q * scale
    w = np.exp(x - x.max())
    p = w / w.sum()
    o = p @ v
    d = (D + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)).max() * abs(scale) + 2.0 ** -39 * np.abs(q).max() * np.abs(k).sum(1).max() * abs(scale)
    rel = 2 * d + 2.0 ** -20 + 2.0 ** -23 + (64 + n / 64) * 2.0 ** -24
    return o, rel * (p @ np.abs(v)) + 2.0 ** -43 / w.sum() * np.abs(v).sum(0) + 2.0 ** -24 * np.abs(o)


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("rows,below", [(1, 17.4), (1, 24.0), (9, 17.4), (1, 10.0)])
def test_float32_small_weights_count(F, code, rows, below):
    """One token takes nearly all the weight, and 32000 tokens far below it the rest: their values are the result, since the
    first one's are zero."""
    n, D, page = 32001, 64, 64
    c = R.Cache([n], heads=1, D=D, page=page, code=code)
    at = 12345
    ids = c.table[0].long()
    c.k.zero_()
    c.ks.fill_(0.01)
    c.k[ids[at // page], 0, at % page] = torch.ones(D).to(code)
    c.v[:] = (torch.rand(c.v.shape, generator=torch.Generator().manual_seed(1)) * 60 + 60).round().to(code)
    c.v[ids[at // page], 0, at % page] = torch.zeros(D).to(code)
    c.vs.fill_(0.01)
    q = torch.full((rows, 1, D), below / (0.01 * D * D ** -0.5))  # the token's score is `below`, all others' 0
    got = F.attention_kv8(q.cuda(), *c.cuda(), None, c.lens.cuda(), causal=False).cpu().double().numpy()
    k, v = c.tokens(0)
    o, tol = _float32_bound(k[:, 0], v[:, 0], q[0, 0].double().numpy(), D ** -0.5)
    off = np.abs(got[:, 0] - o) - tol
    assert (off <= 0).all(), (float(off.max()), float(np.abs(got[:, 0] - o).max() / np.abs(o).max()))


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 12, 2.0 ** 16, 2.0 ** -120, 2.0 ** 127])
def test_float32_queries_with_an_outlier(F, code, size):
    """A query's largest number meets keys that are zero there: the scores are those of the small numbers."""
    n, D, page = 700, 64, 32
    c = R.Cache([n], heads=1, D=D, page=page, code=code)
    c.k[..., 5] = torch.zeros(c.k.shape[:-1]).to(code)
    q = torch.randn(3, 2, D, generator=torch.Generator().manual_seed(2))
    q[..., 5] = size * 1.3
    if size > 2.0 ** 100:
        q[..., 5] = 3.0e38
        q[..., :5] *= 2.0 ** 100
        q[..., 6:] *= 2.0 ** 100
        c.ks *= 2.0 ** -100
    if size < 2.0 ** -100:
        q *= 2.0 ** -118
        q[..., 5] = 2.0 ** -118
        c.ks *= 2.0 ** 118
    got = F.attention_kv8(q.cuda(), *c.cuda(), None, c.lens.cuda(), causal=False).cpu().double().numpy()
    k, v = c.tokens(0)
    for r in range(3):
        for h in range(2):
            o, tol = _float32_bound(k[:, 0], v[:, 0], q[r, h].double().numpy(), D ** -0.5)
            off = np.abs(got[r, h] - o) - tol
            assert (off <= 0).all(), (r, h, float(off.max()), float(np.abs(got[r, h] - o).max() / np.abs(o).max()))


# ------------------------------------------------------------------------------------------ prompts and value scales
@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 26, 2.0 ** 32])
def test_prompts_rows_owe_nothing_to_pages_they_do_not_see(F, code, D, page, window, factor):
    """One page's values are up to 2^32 times the others': rows before it, and rows whose window has left it, are
    as exact as without it.

    The rows that do see it: the kernel feeds the products of weight and value scale, p_j s_j, as float16 numbers of 2^7 at
    least for the row's largest. Where such a number is a subnormal it is off by half a step of 2^-24, which is 2^-32 of
    the largest; with the codes c_j the sum is off by 2^-32 max_j(p_j s_j) sum_j |c_j| at most, on top of what R.attention
    counts. That matters for values whose code is zero in the large page. The other rows get none of it.
    """
    new, G = [270], 4
    heads = _heads(new, G, D)
    c = R.Cache([300], heads=heads, D=D, page=page, code=code)
    big = 128 // page if not window else 64 // page
    c.vs[:] = 20000.0 / R.LIMIT[code] / factor
    c.vs[c.table[0, big]] = 20000.0 / R.LIMIT[code]
    q = torch.randn(270, G * heads, D, generator=torch.Generator().manual_seed(270 + G * heads)).half()
    want, tol = R.attention(c, q, _cu(new), window=window)
    free = np.zeros(270, bool)
    if window:
        free[(big + 1) * page + window - 1 - 30:] = True  # rows are the positions from 30 on
        free[:max(0, big * page - 30)] = True
    else:
        free[:big * page - 30] = True
    ids = c.table[0, :-(-300 // page)].long()
    codes = np.abs(c.v[ids].float().double().transpose(1, 2).reshape(-1, heads, D)[:300].numpy())
    scale = c.vs[ids].double().repeat_interleave(page, 0)[:300].numpy()
    keys, _ = c.tokens(0)
    for row in np.flatnonzero(~free):
        pos = row + 30
        lo = max(0, pos - window + 1) if window else 0
        for h in range(G * heads):
            x = keys[lo:pos + 1, h // G] @ q[row, h].double().numpy() * D ** -0.5
            p = np.exp(x - x.max())
            p /= p.sum()
            tol[row, h] += 2.0 ** -32 * (p * scale[lo:pos + 1, h // G]).max() * codes[lo:pos + 1, h // G].sum(0)
    got = F.attention_kv8(q.cuda(), *c.cuda(), _cu(new).cuda(), c.lens.cuda(), window=window).cpu().double().numpy()
    assert F.device_error(0) == 0 and np.isfinite(got).all()
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), (float(off.max()), float(off[free].max()))
    assert free.sum() > 60 and (np.abs(got[free]) > 0).any(-1).all()


# ------------------------------------------------------------------------------------------ devices
def test_workspace_is_asked_for_on_the_tensors_device(F, monkeypatch):
    """The workspace's size depends on the device's number of SMs: it is asked for, like the launch, with the tensors' device
    current, whichever was current before."""
    at, seen = [0], []  # the current device; the tensors' is 3 (CPU tensors stand in for its)

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            at.append(self.index)

        def __exit__(self, *a):
            at.pop()

    class Library:
        def xrgpu_kv8_attention_workspace_size(self, p, need):
            seen.append(("size", at[-1]))
            need._obj.value = 1000 + at[-1]
            return 0

        def xrgpu_kv8_attention(self, p, ws, nbytes, stream):
            seen.append(("launch", at[-1], nbytes, stream))
            return 0

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[-1])
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 3)
    monkeypatch.setattr(F, "_current_stream", lambda index: 100 + index)
    monkeypatch.setattr(F._native, "load", lambda: Library())
    c = R.Cache([5], heads=1, D=64, page=16, code=INT8)
    for current in (0, 3):
        at[:] = [current]
        seen.clear()
        F.attention_kv8(torch.zeros(1, 2, 64), c.k, c.v, c.ks, c.vs, c.table, None, c.lens)
        assert seen == [("size", 3), ("launch", 3, 1003, 103)] and at == [current]


# ------------------------------------------------------------------------------------------ every form of the kernels
def _form(tokens, seqs, hq, hkv, D, f16, uniform, table_tokens):
    """The kernels that a call takes, by the rules of mmnb_kv8_attn.cu and mmnb_kv8_attn_mma.cuh."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    G, mean = hq // hkv, -(-tokens // seqs)
    rows, pairs = mean * G, seqs * hkv
    prompt = f16 and rows > 64 and pairs * rows * D >= -(-pairs * -(-rows // 256) // sms) * 6500 * 128
    forms = {"prompt"} if prompt else set()
    if prompt and uniform:
        return forms
    slots = -(-(tokens // seqs * G) // 8) * seqs if uniform else tokens * G // 8 + seqs
    split = 8
    while split > 1 and slots * hkv * split > sms:
        split //= 2
    if split > 1 and -(-table_tokens // 32) <= 48 * split:
        return forms | {"cluster"}
    return forms | {"one tile" if min(rows, 64 if prompt else rows) <= 8 else "two tiles"}


def _gpu_cache(lens, hkv, D, page, code, seed):
    """Tensors of a cache in use, made on the GPU: codes of every value, pages in no order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    order = torch.randperm(P, generator=g, device="cuda").int().cpu()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n

    def side():
        codes = torch.randint(-127, 128, (P, hkv, page, D), generator=g, device="cuda", dtype=torch.int8)
        return (codes if code == INT8 else (codes.float() * 3.5).to(E4M3)), (torch.rand(P, hkv, generator=g, device="cuda") * 1.5 + 0.5) * 3.5 / R.LIMIT[code]

    (k, ks), (v, vs) = side(), side()
    return k, v, ks, vs, table.cuda()


def _check_on_gpu(F, dev, lens, new, hq, dtype, seed):
    """As _check, with R.attention's values and tolerance (causal, no window) computed on the GPU in float64, and for int8 codes
    under float16 rows one term more, which matters where every code that a row sees is (next to) zero: the split kernel
    sums p (c + 128) and takes 128 p out again, in four accumulations a step of 32 tokens, each rounded (or truncated: 2^-23) at
    no more than 255 times the sum of the step's weights; times the page's scale s and over all steps that is
    4 * 255 * 2^-23 < 2^-13 of sum_j p_j s_j: 2^-13 of a code."""
    k, v, ks, vs, table = dev
    hkv, page, D = k.shape[1], k.shape[2], k.shape[3]
    G, T = hq // hkv, sum(new)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(T, hq, D, generator=g, device="cuda").to(dtype)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = F.attention_kv8(q, *dev, _cu(new).cuda(), n)
    again = F.attention_kv8(q, *dev, _cu(new).cuda(), n)
    assert F.device_error(0) == 0 and torch.equal(got, again)
    f16, at = dtype == torch.float16, 0
    for b, (total, m) in enumerate(zip(lens, new)):
        if m == 0:
            continue
        rows = slice(at, at + m)
        at += m
        if total == 0:
            assert not got[rows].any()
            continue
        ids = table[b, :-(-total // page)].long()
        kk, vv = ((c[ids].float().double() * s[ids].double()[..., None, None]).transpose(1, 2).reshape(-1, hkv, D)[:total].transpose(0, 1) for c, s in ((k, ks), (v, vs)))
        x = q[rows].double().view(m, hkv, G, D).permute(1, 2, 0, 3).reshape(hkv, G * m, D)
        hide = torch.arange(total, device="cuda") > (total - m + torch.arange(m, device="cuda").repeat(G))[:, None]
        s = (x @ kk.transpose(1, 2) * D ** -0.5).masked_fill(hide, float("-inf"))
        blind = torch.isinf(s.amax(-1))
        w = torch.exp(s - s.amax(-1, keepdim=True)).nan_to_num(0.0)
        sums = w.sum(-1, keepdim=True).clamp(min=1e-300)
        o = (w @ vv) / sums
        d = (D + 8) * 2.0 ** -24 * (x.abs() @ kk.abs().transpose(1, 2)).masked_fill(hide, 0.0).amax(-1, keepdim=True) * D ** -0.5
        rel = 2 * d + 2.0 ** -20 + 2 * (2.0 ** -11 if f16 else 2.0 ** -21) + (64 + total / 64) * 2.0 ** -24
        tol = rel * (w @ vv.abs()) / sums + 2.0 ** -25 / sums * ((~hide).double() @ vv.abs()) + (2.0 ** -11 if f16 else 2.0 ** -24) * o.abs() + 2.0 ** -24 * f16
        if f16 and k.dtype == INT8:
            tol = tol + 2.0 ** -13 * (w @ vs[ids].double().repeat_interleave(page, 0)[:total].t()[..., None]) / sums
        mine = got[rows].double().view(m, hkv, G, D).permute(1, 2, 0, 3).reshape(hkv, G * m, D)
        off = ((mine - o).abs() - tol).masked_fill(blind[..., None], 0.0)
        assert bool((off <= 0).all()), (b, float(off.max()))
        assert not mine[blind].any()
    return got


LONG = [("one tile", 1, 4), ("two tiles", 3, 4), ("two tiles", 1, 24)]  # form, rows a sequence, group


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (64, 128), (128, 32)])
@pytest.mark.parametrize("form,rows,G", LONG)
def test_long_runs_of_the_split_kernel(F, code, dtype, D, page, form, rows, G):
    """Runs of more than 16 steps a warp (rings used again and again, page ids looked up in several batches), segments cut between
    CTAs, sequences of very different lengths."""
    hkv = 8
    rng = np.random.default_rng(page)
    lens = [int(n) for n in rng.integers(3000, 9000, 40)] + [rows, 31 + rows, 64]
    new = [rows] * len(lens)
    assert _form(sum(new), len(new), G * hkv, hkv, D, dtype == torch.float16, False, -(-max(lens) // page) * page) == {form}
    assert sum(-(-n // 32) for n in lens) * hkv * -(-rows * G // (8 if form == "one tile" else 16)) > 20 * 6 * 2 * 148
    _check_on_gpu(F, _gpu_cache(lens, hkv, D, page, code, D + page), lens, new, G * hkv, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_forms_are_all_reached(F, dtype):
    """A few sequences of each form by its rule: the same call shapes as in the tests above, counted."""
    seen = set()
    for lens, new, hkv, G, D in (([2000], [1], 2, 4, 128), ([700] * 30, [1] * 30, 8, 4, 64), ([700] * 30, [5] * 30, 8, 4, 64), ([900, 20], [400, 1], 8, 4, 128),
                                 ([900, 700], [400, 400], 8, 4, 128)):
        seen |= (form := _form(sum(new), len(new), G * hkv, hkv, D, dtype == torch.float16, False, -(-max(lens) // 64) * 64))
        assert form
        _check_on_gpu(F, _gpu_cache(lens, hkv, D, 64, INT8, 3), lens, new, G * hkv, dtype, 2)
    assert seen == {"cluster", "one tile", "two tiles"} | ({"prompt"} if dtype == torch.float16 else set())


def _many(count, most, seed):
    """(tokens held before, new rows) of `count` short ragged sequences, empty ones among them."""
    rng = np.random.default_rng(seed)
    past, new = rng.integers(0, 120, count), rng.integers(0, most + 1, count)
    past[::7] = 0
    new[::5] = 0
    new[count // 2: count // 2 + 40] = 0
    return past.tolist(), new.tolist()


@gpu
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("count,most", [(130, 3), (400, 1), (700, 40)])
def test_many_sequences_append_and_read(F, code, count, most):
    """More sequences than a CTA has threads: the searches go on past their first pass."""
    past, new = _many(count, most, count)
    c = R.Cache([a + b for a, b in zip(past, new)], heads=2, D=64, page=16, code=code, seed=count)
    c.poison_tails()
    T = sum(new)
    k, v = (torch.randn(T + 3, 2, 64, generator=torch.Generator().manual_seed(i)) * 3 for i in (1, 2))
    cu, dev = _cu(new), c.cuda()
    F.kv8_append(k.cuda(), v.cuda(), *dev, cu.cuda(), c.lens.cuda())
    R.append(c, k, v, cu)
    used = c.table[c.table >= 0].long()
    assert torch.equal(dev[2].cpu()[used], c.ks[used]) and torch.equal(dev[3].cpu()[used], c.vs[used])
    rk, rv = F.kv8_read(*dev, cu.cuda(), c.lens.cuda(), rows=T + 3, dtype=torch.float32)
    want = [torch.from_numpy(np.concatenate([c.tokens(b)[i][past[b]:] for b in range(count)])).float() for i in (0, 1)]
    for got, w in ((rk, want[0]), (rv, want[1])):
        assert torch.equal(got[:T].cpu(), w) and not got[T:].any()
    assert F.device_error(0) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("count,most,hkv,form", [(400, 1, 2, {"one tile"}), (700, 7, 1, {"two tiles"}), (90, 150, 2, {"prompt", "two tiles"})])
def test_many_sequences_attention(F, dtype, count, most, hkv, form):
    past, new = _many(count, most, count)
    lens = [max(1, a + b) if b else a + b for a, b in zip(past, new)]
    if dtype == torch.float16 or "prompt" not in form:
        assert _form(sum(new), count, 4 * hkv, hkv, 128, dtype == torch.float16, False, -(-max(lens) // 16) * 16) == form
    _check_on_gpu(F, _gpu_cache(lens, hkv, 128, 16, INT8, count), lens, new, 4 * hkv, dtype, 3)
