"""quantize_int8 and int8_matmul (ops.py) against their definition in float64.

Codes: rne(127 x / max) in float64; for bf16 rows they have to be equal (a
quotient is either a border, met exactly, or at least 2^-9 away from one), for
fp32 rows within 2^-20 of a border either neighbour is right.  Products: the
int32 sum is exact; its conversion to fp32 and the two scales round by at most
2^-24 each (1e-6 relative bounds the four with room for the scale's own
rounding), then one rounding to bf16 (2^-8)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _define(x):
    """(codes before rounding, scale) in float64."""
    a = np.abs(x).max(axis=-1, keepdims=True)
    with np.errstate(all="ignore"):
        v = np.where(a > 0, 127.0 * x / a, 0.0)
    return v, a[..., 0] / 127.0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 0), (5, 64, 8), (2, 255, 3), (9, 1000, 0), (4, 14336, 0),
                                           (2, 20001, 0)])
def test_quantize(moe, dtype, rows, cols, pad):
    print(f"quantize {dtype} {rows}x{cols}+{pad}", flush=True)
    rng = np.random.default_rng([rows, cols])
    t = torch.full((rows, cols + pad), float("nan"), dtype=DT[dtype])
    t[:, :cols] = torch.from_numpy(rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-3, 4, (rows, 1))).to(DT[dtype])
    x = t.cuda()[:, :cols]
    q, s = moe.quantize_int8(x)
    v, sc = _define(t[:, :cols].double().numpy())
    got = q.cpu().numpy().astype(np.float64)
    if dtype == "bf16":
        assert np.array_equal(got, np.round(v))
    else:
        assert (np.abs(got - v) <= 0.5 + 2.0**-20).all()
    assert np.allclose(s.cpu().numpy(), sc, rtol=2.0**-23, atol=0)


def test_quantize_borders_and_special_rows(moe):
    # odd multiples of max / 254 are borders: half to even
    n = np.arange(-254, 255, dtype=np.float32)
    x = torch.from_numpy(np.stack([n, n * 2.0**100, n * 2.0**-100])).cuda()
    q, _ = moe.quantize_int8(x)
    assert all(np.array_equal(r, np.round(n / 2)) for r in q.cpu().numpy())
    q, _ = moe.quantize_int8(x.to(torch.bfloat16))
    assert np.array_equal(q.cpu().numpy()[0], np.round(n / 2))
    x = torch.zeros(8, 300)
    x[1, 7], x[2, 299] = float("inf"), float("nan")
    x[3, :] = 3e38
    x[4, 5] = 1e-45
    x[5, 0], x[5, 1] = -1e-38, 1e-45
    x[6] = torch.linspace(-3.4e38, 3.4e38, 300)
    q, s = (t.cpu().numpy() for t in moe.quantize_int8(x.cuda()))
    assert s[0] == 0 and (q[0] == 0).all()
    assert np.isnan(s[1]) and np.isnan(s[2]) and (q[1] == 0).all() and (q[2] == 0).all()
    assert (q[3] == 127).all() and q[4, 5] == 127 and q[5, 0] == -127 and q[5, 1] == 0
    # linspace forms end - start = 6.8e38, past fp32: row 6 holds values that are not finite
    assert not torch.isfinite(x[6]).all() and np.isnan(s[6]) and (q[6] == 0).all()
    v = torch.linspace(-1, 1, 300) * 3.4e38  # 127 v overflows, v does not
    q, s = (t.cpu().numpy() for t in moe.quantize_int8(v[None].cuda()))
    ref = np.round(127.0 * v.double().numpy() / v.abs().max().double().item())
    assert np.isfinite(s).all() and np.abs(q[0] - ref).max() <= 1 and q[0, 0] == -127 and q[0, -1] == 127
    w = torch.randn(4, 6, 50, device="cuda")
    q, s = moe.quantize_int8(w)  # a weight: a scale per output channel
    q2, s2 = moe.quantize_int8(w.reshape(24, 50))
    assert q.shape == w.shape and s.shape == (4, 6) and torch.equal(q.reshape(24, 50), q2) and torch.equal(s.reshape(-1), s2)


# group lengths, K, N: streamed and tiled forms, odd sizes, long sums
SHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([2], 4096, 130),
    ([17, 0, 1, 64], 128, 96),
    ([33, 130, 5, 0, 300], 208, 136),
    ([16, 16, 40, 2], 129, 257),
    ([100, 90, 65], 333, 72),
    ([700, 0, 900, 500], 144, 2048),
    ([3000, 5500], 160, 4112),
    ([40, 30], 20000, 33),
]


@pytest.mark.parametrize("wpad", [0, 5])
@pytest.mark.parametrize("xt,odt", [("bf16", "bf16"), ("f32", "f32"), ("codes", "f32")])
def test_int8_matmul(moe, xt, odt, wpad):
    for lens, K, N in SHAPES:
        print(f"int8 {xt}->{odt} wpad={wpad} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, wpad])
        M, E, tail = sum(lens), len(lens), 2
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        wb = torch.full((E, N, K + wpad), 99, dtype=torch.int8)
        wb[:, :, :K] = torch.from_numpy(rng.integers(-127, 128, (E, N, K)).astype(np.int8))
        w = wb.cuda()[:, :, :K]
        ws = torch.from_numpy(rng.uniform(0.001, 0.02, (E, N)).astype(np.float32)).cuda()
        if xt == "codes":
            q = rng.integers(-128, 128, (M + tail, K)).astype(np.int8)
            s = rng.uniform(0.001, 0.02, M + tail).astype(np.float32)
            kw = dict(x_scale=torch.from_numpy(s).cuda())
            x = torch.from_numpy(q).cuda()
        else:
            x = torch.from_numpy(rng.standard_normal((M + tail, K))).to(DT[xt]).cuda()
            tq, ts = moe.quantize_int8(x)
            q, s, kw = tq.cpu().numpy(), ts.cpu().numpy(), {}
        out = torch.full((M + tail, N), 776.0, dtype=DT[odt], device="cuda")
        moe.int8_matmul(x, w, ws, off, out=out, **kw)
        got, W, at = out.cpu().double().numpy(), wb[:, :, :K].numpy().astype(np.float64), 0
        for e, n in enumerate(lens):
            r = slice(at, at + n)
            ref = (q[r].astype(np.float64) @ W[e].T) * s[r, None].astype(np.float64) * ws[e].cpu().double().numpy()
            tol = np.abs(ref) * (1e-6 + (2.0**-8 if odt == "bf16" else 0.0)) + 1e-37
            assert (np.abs(got[r] - ref) <= tol).all(), float(np.abs(got[r] - ref).max())
            at += n
        assert (got[M:] == 776.0).all()


def test_extreme_sums_are_exact(moe):
    # the largest int32 sum the entry allows, of one sign
    K = 131071
    for rows in (1, 40):
        x = torch.full((rows, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((17, K), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(rows, device="cuda")
        y = moe.int8_matmul(x, w, torch.ones(17, device="cuda"), x_scale=one, out_dtype=torch.float32)
        assert (y == float(128 * 128 * K)).all()


def test_nan_rows_and_graph(moe):
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((70, 256))).to(torch.bfloat16).cuda()
    w, ws = moe.quantize_int8(torch.from_numpy(rng.standard_normal((2, 80, 256)).astype(np.float32)).cuda())
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    want = [moe.int8_matmul(x * f, w, ws, off) for f in (1, 3, -2)]
    buf = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.int8_matmul(buf, w, ws, off)
    for i, f in enumerate((1, 3, -2)):
        buf.copy_(x * f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
    x[4, 9], x[50, 1] = float("nan"), float("-inf")
    fin = torch.isfinite(moe.int8_matmul(x, w, ws, off)).all(dim=1)
    assert not fin[4] and not fin[50] and fin.sum() == 68


def test_split_sums_with_empty_groups(moe):
    # long sums of few rows: k split over workgroups, the fold finds each row's
    # group among empty ones (first, middle, last) and groups outside the rows
    rng = np.random.default_rng(15)
    for lens, start, K, N in (([0, 0, 2, 0, 1, 0, 0], 0, 20000, 17), ([0, 40, 0, 0, 31, 0], 3, 9000, 64)):
        print(f"int8 split lens={lens} K={K} N={N}", flush=True)
        E, M = len(lens), sum(lens)
        q = torch.from_numpy(rng.integers(-127, 128, (M + start + 2, K)).astype(np.int8)).cuda()
        w = torch.from_numpy(rng.integers(-127, 128, (E, N, K)).astype(np.int8)).cuda()
        xs, ws = (torch.from_numpy(rng.uniform(0.5, 2, s).astype(np.float32)).cuda() for s in ((M + start + 2,), (E, N)))
        off = torch.tensor(np.concatenate([[start], start + np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        y = moe.int8_matmul(q, w, ws, off, x_scale=xs, out_dtype=torch.float32).cpu().double().numpy()
        Q, W = q.cpu().numpy().astype(np.int64), w.cpu().numpy().astype(np.int64)
        XS, WS = xs.cpu().double().numpy(), ws.cpu().double().numpy()
        at = start
        for e, n in enumerate(lens):
            s = slice(at, at + n)
            ref = (Q[s] @ W[e].T) * XS[s, None] * WS[e]
            # the exact sum to fp32 and two products: three roundings
            assert (np.abs(y[s] - ref) <= 3.01 * 2.0**-24 * np.abs(ref)).all(), e
            at += n
        assert (y[:start] == 0).all() and (y[at:] == 0).all()


@pytest.mark.parametrize("pad", [0, 4])
def test_codes_of_whole_dwords(moe, pad):
    # code rows of a multiple of four that do not start on 16 bytes; the padding
    # holds codes that must not be summed
    rng = np.random.default_rng(18)
    for lens, K, N in (([20, 0, 45], 4, 30), ([33, 130, 0, 300], 204, 134), ([700, 0, 900], 68, 2046), ([90], 5444, 62)):
        print(f"int8 dword rows pad={pad} lens={lens} K={K} N={N}", flush=True)
        E, M = len(lens), sum(lens)
        q = torch.from_numpy(rng.integers(-127, 128, (M, K + pad)).astype(np.int8)).cuda()[:, :K]
        w = torch.from_numpy(rng.integers(-127, 128, (E, N, K + pad)).astype(np.int8)).cuda()[:, :, :K]
        xs, ws = torch.ones(M, device="cuda"), torch.ones(E, N, device="cuda")
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        y = moe.int8_matmul(q, w, ws, off, x_scale=xs, out_dtype=torch.float32).cpu().double().numpy()
        Q, W, at = q.cpu().numpy().astype(np.int64), w.cpu().numpy().astype(np.int64), 0
        for e, n in enumerate(lens):
            ref = Q[at:at + n] @ W[e].T
            assert (np.abs(y[at:at + n] - ref) <= 2.0**-24 * np.abs(ref)).all(), e
            at += n


# streamed, tiled, k split (streamed and tiled): each has its own last step
SCALED = [([3, 0, 2], 64, 40), ([40, 30, 0, 90], 96, 72), ([3, 0, 2], 20000, 17), ([40, 30], 20000, 33)]


@pytest.mark.parametrize("odt", ["f32", "bf16"])
def test_scales_far_from_one(moe, odt):
    # rows and channels whose scales nearly cancel: no step on the way may leave
    # fp32's range or lose bits to its subnormals where the result does not
    for lens, K, N in SCALED:
        print(f"int8 far scales ->{odt} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, 21])
        E, M = len(lens), sum(lens)
        q = torch.from_numpy(rng.integers(64, 128, (M, K)).astype(np.int8)).cuda()
        w = torch.from_numpy(rng.integers(64, 128, (E, N, K)).astype(np.int8)).cuda()
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        Q, W = q.cpu().numpy().astype(np.int64), w.cpu().numpy().astype(np.int64)
        for xs, ws in ((1e33, 1e-33), (3e38, 1e-40), (1e-37, 1e30), (1e-43, 1e36), (-2e35, 1e-36), (1.0, 1.0), (0.0, 2.0)):
            sx = torch.full((M,), xs, device="cuda") * torch.linspace(0.5, 1.0, M, device="cuda")
            sw = torch.full((E, N), ws, device="cuda")
            y = moe.int8_matmul(q, w, sw, off, x_scale=sx, out_dtype=DT[odt]).cpu().double().numpy()
            SX, SW, at = sx.cpu().double().numpy(), sw.cpu().double().numpy(), 0
            for e, n in enumerate(lens):
                s = slice(at, at + n)
                ref = (Q[s] @ W[e].T) * SX[s, None] * SW[e]
                # the exact sum to fp32 and two products, then the result's type
                tol = (3.01 * 2.0**-24 + (2.0**-8 if odt == "bf16" else 0.0)) * np.abs(ref)
                assert np.isfinite(ref).all() and (np.abs(y[s] - ref) <= tol).all(), (xs, ws, e)
                at += n


@pytest.mark.parametrize("xt", ["bf16", "f32"])
def test_rows_far_from_one(moe, xt):
    # the same through the call's own quantiser
    rng = np.random.default_rng(22)
    x = torch.from_numpy(rng.standard_normal((6, 300)).astype(np.float32))
    x = (x * torch.tensor([1e33, 1e-34, 1.0, 1e35, 1e-30, 1e37])[:, None]).to(DT[xt]).cuda()
    w = torch.from_numpy(rng.integers(-127, 128, (33, 300)).astype(np.int8)).cuda()
    q, s = moe.quantize_int8(x)
    for ws in (1e-6, 1e-2, 1.0):
        y = moe.int8_matmul(x, w, torch.full((33,), ws, device="cuda"), out_dtype=torch.float32).cpu().double().numpy()
        sw = float(np.float32(ws))
        ref = (q.cpu().numpy().astype(np.int64) @ w.cpu().numpy().astype(np.int64).T) * s.cpu().double().numpy()[:, None] * sw
        big = np.abs(ref) > 3.4e38
        assert (np.abs(y - ref) <= 3.01 * 2.0**-24 * np.abs(ref) + 2.0**-149)[~big].all() and np.isinf(y[big]).all()


def test_scales_that_are_not_finite(moe):
    # a NaN scale gives NaN, an infinite one an infinity, in their rows and columns only
    rng = np.random.default_rng(23)
    for M, K, N in ((4, 64, 20), (90, 64, 70), (3, 20000, 17)):
        q = torch.from_numpy(rng.integers(1, 128, (M, K)).astype(np.int8)).cuda()
        w = torch.from_numpy(rng.integers(1, 128, (N, K)).astype(np.int8)).cuda()
        xs, ws = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
        xs[1], xs[2], ws[3], ws[5] = float("nan"), float("inf"), float("nan"), float("-inf")
        y = moe.int8_matmul(q, w, ws, x_scale=xs, out_dtype=torch.float32).cpu().numpy()
        assert np.isnan(y[1]).all() and np.isnan(y[:, 3]).all()
        rest = np.delete(np.arange(N), [3, 5])
        assert np.isposinf(y[2, rest]).all() and np.isneginf(np.delete(y[:, 5], 1)).all()
        assert np.isfinite(y[np.ix_([0, M - 1], rest)] if M > 3 else y[0, rest]).all()


@pytest.mark.parametrize("odt", ["f32", "bf16"])
def test_scales_far_from_one(moe, odt):
    # rows and channels whose scales nearly cancel: no step on the way may leave
    # fp32's range or lose bits to its subnormals where the result does not
    for lens, K, N in SCALED:
        print(f"int8 far scales ->{odt} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, 21])
        E, M = len(lens), sum(lens)
        q = torch.from_numpy(rng.integers(64, 128, (M, K)).astype(np.int8)).cuda()
        w = torch.from_numpy(rng.integers(64, 128, (E, N, K)).astype(np.int8)).cuda()
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        Q, W = q.cpu().numpy().astype(np.int64), w.cpu().numpy().astype(np.int64)
        for xs, ws in ((1e33, 1e-33), (3e38, 1e-40), (1e-37, 1e30), (1e-43, 1e36), (-2e35, 1e-36), (1.0, 1.0), (0.0, 2.0)):
            sx = torch.full((M,), xs, device="cuda") * torch.linspace(0.5, 1.0, M, device="cuda")
            sw = torch.full((E, N), ws, device="cuda")
            y = moe.int8_matmul(q, w, sw, off, x_scale=sx, out_dtype=DT[odt]).cpu().double().numpy()
            SX, SW, at = sx.cpu().double().numpy(), sw.cpu().double().numpy(), 0
            for e, n in enumerate(lens):
                s = slice(at, at + n)
                ref = (Q[s] @ W[e].T) * SX[s, None] * SW[e]
                # the exact sum to fp32 and two products, then the result's type
                tol = (3.01 * 2.0**-24 + (2.0**-8 if odt == "bf16" else 0.0)) * np.abs(ref)
                assert np.isfinite(ref).all() and (np.abs(y[s] - ref) <= tol).all(), (xs, ws, e)
                at += n

@pytest.mark.parametrize("lens,K,N", [([700, 0, 900, 500], 144, 2048), ([3000, 5500], 160, 4112)])
def test_far_scales_in_large_tiles(moe, lens, K, N):
    # 128 x 128 and 256 x 256 tiles that hold one row of a far scale, many, or none
    print(f"int8 far scales in large tiles lens={lens}", flush=True)
    rng = np.random.default_rng([K, N, 24])
    E, M = len(lens), sum(lens)
    q = torch.from_numpy(rng.integers(64, 128, (M, K)).astype(np.int8)).cuda()
    w = torch.from_numpy(rng.integers(64, 128, (E, N, K)).astype(np.int8)).cuda()
    sx, sw = torch.ones(M, device="cuda"), torch.full((E, N), 1e-3, device="cuda")
    sx[5], sx[300:310], sx[600], sx[M - 1], sx[M - 2] = 1e35, 1e-42, 0.0, 3e38, -1e-40
    sw[:, 3::7] = 1e-36
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    y = moe.int8_matmul(q, w, sw, off, x_scale=sx, out_dtype=torch.float32).double()
    at = 0
    for e, n in enumerate(lens):
        s = slice(at, at + n)
        ref = (q[s].double() @ w[e].double().t().contiguous()) * sx[s, None].double() * sw[e].double()
        # three roundings, the last one possibly to a subnormal; past fp32's largest: infinity
        big = ref.abs() > 3.4028236e38
        assert ((y[s] - ref).abs() <= 3.01 * 2.0**-24 * ref.abs() + 2.0**-149)[~big].all(), e
        assert torch.isinf(y[s])[big].all() and (big.any() or e != E - 1)
        at += n


@pytest.mark.parametrize("rows", [2**20 + 9, 2**23 + 5])
def test_millions_of_rows(moe, rows):
    # more rows than one dimension of a launch takes, through the quantiser and the product
    print(f"int8 rows {rows}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 16, generator=g, device="cuda").to(torch.bfloat16)
    q, s = moe.quantize_int8(x)
    most = x.abs().amax(1, keepdim=True).double()
    assert torch.equal(q.double(), torch.round(127 * x.double() / most))
    assert torch.equal(s, (most[:, 0] / 127).float())
    w, ws = moe.quantize_int8(torch.randn(24, 16, generator=g, device="cuda"))
    y = moe.int8_matmul(x, w, ws, out_dtype=torch.float32)
    part = slice(rows - 70, rows)
    ref = (q[part].double() @ w.double().t()) * s[part, None].double() * ws.double()
    assert ((y[part].double() - ref).abs() <= 3.01 * 2.0**-24 * ref.abs()).all()
    head = (q[:70].double() @ w.double().t()) * s[:70, None].double() * ws.double()
    assert ((y[:70].double() - head).abs() <= 3.01 * 2.0**-24 * head.abs()).all()
