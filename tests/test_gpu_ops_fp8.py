"""quantize_fp8 and fp8_matmul (ops.py) against their definition in float64.

Codes: the e4m3 value nearest to 448 x / max|block| (half: the even code), decided in
integers; they have to be equal.  Scales: one division in fp32, half a step (2^-24).

Products: a block's 128 products, summed in fp32, then times the product of its two
scales (rounded, 2^-24) and added to the fp32 sum of the blocks: at most (K + 4) 2^-23 of
the sum of the magnitudes, then one rounding to the result's type, half a step: 2^-8 of a
bf16 value, 2^-24 of an fp32 one.

bf16 results of tiles (more rows than are streamed) come from the matrix unit's 8-bit
instruction, which cuts the products of 8 neighbours along k to a grid of 2^-13 times the
power of two of the largest (in tests of one large and one small product: 2^-13 of it is
kept, 2^-14 is not).  The largest itself has 6 bits below its leading one and lies on the
grid; each of the seven others loses less than 2^-13 of the largest, which is at most the
sum of the eight magnitudes: less than 7 * 2^-13 of the sum of all magnitudes."""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SENTINEL = 776.0  # exact in bf16 and fp32
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = {"bf16": 2.0**-8, "f32": 2.0**-24}
F8 = torch.float8_e4m3fn
# the finite codes 0 .. 126 and their values
VALUES = np.array([m * 2.0**-9 if e == 0 else (8 + m) * 2.0**(e - 10) for e in range(16) for m in range(8)][:127])


def _spread(s, rows, cols, block_rows):
    """A block's scale at each of its elements."""
    return np.repeat(np.repeat(s, block_rows, axis=-2)[..., :rows, :], 128, axis=-1)[..., :cols]


def _blocks_max(x, block_rows):
    *lead, rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    p = np.zeros((*lead, rb * block_rows, cb * 128))
    p[..., :rows, :cols] = np.abs(x)
    return p.reshape(*lead, rb, block_rows, cb, 128).max(axis=(-3, -1))


def _define(x, block_rows):
    """(codes' values, scales) of (..., rows, cols) in float64: 448 |x| against border * max,
    both exact there (27 bits, and 5 of a border times 24)."""
    top = _blocks_max(x, block_rows)
    m = _spread(top, x.shape[-2], x.shape[-1], block_rows)
    v = 448.0 * np.abs(x)
    code = np.zeros(x.shape, dtype=np.int64)
    for k in range(126):
        border = (VALUES[k] + VALUES[k + 1]) / 2 * m
        code += (v > border) | ((v == border) & (k % 2 == 1))
    return np.where(m > 0, np.copysign(VALUES[code], x), 0.0), top / 448.0


def _f64(t):
    return t.detach().cpu().float().double().numpy()


def _check_codes(x, q, s, block_rows, what):
    """x as (..., rows, cols) numpy."""
    want, scale = _define(x, block_rows)
    got = _f64(q).reshape(x.shape)
    assert np.array_equal(got, want), (what, int((got != want).sum()))
    assert np.allclose(_f64(s).reshape(scale.shape), scale, rtol=2.0**-24 * 1.001, atol=2.0**-149), what


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 0), (5, 64, 8), (2, 255, 3), (9, 1000, 0), (4, 14336, 0),
                                           (130, 136, 0), (1, 20001, 0), (300, 128, 16)])
def test_quantize_rows(moe, dtype, rows, cols, pad):
    print(f"quantize fp8 {dtype} {rows}x{cols}+{pad}", flush=True)
    rng = np.random.default_rng([rows, cols])
    t = torch.full((rows, cols + pad), float("nan"), dtype=DT[dtype])
    t[:, :cols] = torch.from_numpy(rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-3, 4, (rows, cols))).to(DT[dtype])
    x = t.cuda()[:, :cols]
    q, s = moe.quantize_fp8(x)
    assert q.dtype == F8 and q.shape == x.shape and s.shape == (rows, -(-cols // 128))
    _check_codes(_f64(x), q, s, 1, "rows")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("E,rows,cols,pad", [(1, 1, 1, 0), (3, 5, 7, 1), (2, 128, 128, 0), (2, 129, 127, 0), (3, 260, 392, 8),
                                             (1, 1000, 64, 4)])
def test_quantize_tiles(moe, dtype, E, rows, cols, pad):
    print(f"quantize fp8 128 x 128 {dtype} {E}x{rows}x{cols}+{pad}", flush=True)
    rng = np.random.default_rng([E, rows, cols])
    t = torch.full((E, rows + 2, cols + pad), float("nan"), dtype=DT[dtype])
    t[:, :rows, :cols] = torch.from_numpy(rng.standard_normal((E, rows, cols)) * 10.0 ** rng.integers(-3, 4, (E, rows, cols))).to(DT[dtype])
    x = t.cuda()[:, :rows, :cols]
    q, s = moe.quantize_fp8(x, block_rows=128)
    assert q.shape == x.shape and s.shape == (E, -(-rows // 128), -(-cols // 128))
    _check_codes(_f64(x), q, s, 128, "tiles")
    # blocks of 128 x 128 are those of the transpose
    qt, st = moe.quantize_fp8(x.transpose(1, 2).contiguous(), block_rows=128)
    assert torch.equal(qt.float(), q.float().transpose(1, 2)) and torch.equal(st, s.transpose(1, 2))
    if E == 1:
        q2, s2 = moe.quantize_fp8(x[0], block_rows=128)
        assert torch.equal(q2.float(), q[0].float()) and torch.equal(s2, s[0])
    q3, s3 = moe.quantize_fp8(x)  # rows of a tensor of three dimensions
    _check_codes(_f64(x), q3, s3, 1, "rows of matrices")
    assert s3.shape == (E, rows, -(-cols // 128))


@pytest.mark.parametrize("scale", [1.0, 2.0**100, 2.0**-100, 2.0**-130, 2.0**119, 7.0, 1 / 3])
def test_quantize_borders(moe, scale):
    # every border between two codes, met exactly, and its neighbours in fp32 on both
    # sides; for blocks of any magnitude, maxima that are no power of two among them
    mid = (VALUES[1:] + VALUES[:-1]) / 2
    v = np.concatenate([mid, VALUES]).astype(np.float32)
    v = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf))])
    v = v[v <= 448]
    rows = np.zeros((-(-len(v) // 126), 128), dtype=np.float32)
    for i in range(rows.shape[0]):
        part = v[i * 126:(i + 1) * 126]
        rows[i, 1:1 + len(part)] = part * np.where(np.arange(len(part)) % 2, 1, -1)
    rows[:, 0] = 448
    with np.errstate(over="ignore"):
        rows = (rows * np.float32(scale)).astype(np.float32)
    assert np.isfinite(rows).all()
    q, s = moe.quantize_fp8(torch.from_numpy(rows).cuda())
    _check_codes(rows.astype(np.float64), q, s, 1, scale)


def test_quantize_special_blocks(moe):
    x = torch.zeros(8, 300)
    x[1, 7], x[2, 299] = float("inf"), float("nan")
    x[3, :] = 3e38
    x[4, 5] = 1e-45
    x[5, 0], x[5, 1] = -1e-38, 1e-45
    x[6] = torch.linspace(-1, 1, 300) * 3.4e38
    q, s = moe.quantize_fp8(x.cuda())
    q, s = q.float().cpu(), s.cpu()
    assert (s[0] == 0).all() and (q[0] == 0).all()
    # only the block that holds it
    assert torch.isnan(s[1, 0]) and (q[1, :128] == 0).all() and (s[1, 1:] == 0).all()
    assert torch.isnan(s[2, 2]) and (s[2, :2] == 0).all() and (q[2] == 0).all()
    assert (q[3] == 448).all() and torch.isfinite(s[3]).all()
    assert q[4, 5] == 448 and q[5, 0] == -448 and q[5, 1] == 0
    want, scale = _define(x[6:7].double().numpy(), 1)
    assert np.array_equal(q[6:7].double().numpy(), want)
    q, s = moe.quantize_fp8(x.cuda(), block_rows=128)
    assert torch.isnan(s[0]).tolist() == [True, False, True] and (q[:, :128].float() == 0).all()
    empty, scales = moe.quantize_fp8(torch.zeros(0, 130, device="cuda"))
    assert empty.shape == (0, 130) and scales.shape == (0, 2)


# group lengths, K, N: streamed and tiled forms, odd sizes, long sums
SHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([2], 4096, 130),
    ([17, 0, 1, 64], 128, 96),
    ([33, 130, 5, 0, 300], 208, 136),
    ([16, 16, 40, 2], 129, 257),
    ([100, 90, 65], 333, 72),
    ([33, 90, 65], 388, 200),       # rows of whole dwords
    ([700, 0, 900, 500], 144, 2048),
    ([700, 0, 900, 500], 1168, 520),
    ([40, 30], 20000, 33),
    ([5] * 70, 256, 48),            # more groups than a wave has lanes
]


def _codes(rng, shape):
    """Any finite codes."""
    return torch.from_numpy((rng.integers(0, 127, shape) | (rng.integers(0, 2, shape) << 7)).astype(np.uint8))


def _scales(rng, shape):
    return torch.from_numpy(rng.uniform(0.001, 0.02, shape).astype(np.float32))


def _weights(rng, E, N, K, pad):
    t = torch.full((E, N, K + pad), 0x7F, dtype=torch.uint8)  # NaN behind the rows
    t[:, :, :K] = _codes(rng, (E, N, K))
    return t.cuda().view(F8)[:, :, :K], _scales(rng, (E, -(-N // 128), -(-K // 128))).cuda()


def _check_product(lens, got, q, xs, w, ws, odt, start=0, tiles=True):
    """got: y as numpy; q (M, K) codes with scales; tiles: the call was not streamed."""
    X = _f64(q) * _spread(_f64(xs), q.shape[0], q.shape[1], 1)
    W = _f64(w) * _spread(_f64(ws), w.shape[1], w.shape[2], 128)
    at, K = start, q.shape[1]
    for e, n in enumerate(lens):
        r = slice(at, at + n)
        ref, mag = X[r] @ W[e].T, np.abs(X[r]) @ np.abs(W[e].T)
        cut = 7 * 2.0**-13 if odt == "bf16" and tiles else 0.0
        tol = ((K + 4) * 2.0**-23 + cut) * mag + np.abs(ref) * STEP[odt] + 1e-37
        bad = ~(np.abs(got[r] - ref) <= tol)
        assert not bad.any(), (int(bad.sum()), float(np.abs(got[r] - ref).max()), float(mag.max()))
        at += n


@pytest.mark.parametrize("wpad", [0, 16, 5])
@pytest.mark.parametrize("xt,odt", [("bf16", "bf16"), ("f32", "f32"), ("codes", "f32")])
def test_fp8_matmul(moe, xt, odt, wpad):
    for lens, K, N in SHAPES:
        print(f"fp8 {xt}->{odt} wpad={wpad} lens={lens[:6]} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, wpad])
        M, E, tail = sum(lens), len(lens), 2
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        w, ws = _weights(rng, E, N, K, wpad)
        if xt == "codes":
            x = _codes(rng, (M + tail, K)).cuda().view(F8)
            xs = _scales(rng, (M + tail, -(-K // 128))).cuda()
            q, kw = x, dict(x_scale=xs)
        else:
            x = torch.from_numpy(rng.standard_normal((M + tail, K))).to(DT[xt]).cuda()
            (q, xs), kw = moe.quantize_fp8(x), {}
        out = torch.full((M + tail, N + 3), SENTINEL, dtype=DT[odt], device="cuda")
        y = moe.fp8_matmul(x, w, ws, off, out=out[:, :N], **kw)
        _check_product(lens, _f64(y), q, xs, w, ws, odt)
        assert (_f64(out)[M:] == SENTINEL).all() and (_f64(out)[:, N:] == SENTINEL).all()
        if xt != "codes":  # what the call quantises is what quantize_fp8 gives
            assert torch.equal(moe.fp8_matmul(q, w, ws, off, x_scale=xs, out_dtype=DT[odt])[:M], y[:M])


def test_large_tiles(moe):
    rng = np.random.default_rng(5)
    for lens, K, N in (([3000, 5500], 160, 7168), ([2100, 1, 3000, 3400], 272, 7064)):
        x, xs = _codes(rng, (sum(lens), K)).cuda().view(F8), _scales(rng, (sum(lens), -(-K // 128))).cuda()
        w, ws = _weights(rng, len(lens), N, K, 0)
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        for odt in ("bf16", "f32"):
            res = []
            names = kernels_of(lambda: res.append(moe.fp8_matmul(x, w, ws, off, x_scale=xs, out_dtype=DT[odt])))
            # fp32 results: the codes in bf16, 128 x 128 tiles
            assert (names["op_f8_kernel"][0], names["op_f8_kernel"][7]) == (("256", "false") if odt == "bf16" else ("128", "true"))
            _check_product(lens, _f64(res[0]), x, xs, w, ws, odt)


def test_forms(moe):
    for lens, K, N, tile, split in (([3000, 5500], 160, 7168, "256", False), ([700, 0, 900, 500], 144, 2048, "128", False),
                                    ([33, 130, 5, 0, 300], 208, 136, "64", False), ([40, 30], 20000, 33, "64", True),
                                    ([0, 3, 0], 7, 5, None, False), ([0, 9, 0], 5001, 50, "64", True),
                                    ([0, 0, 2, 0, 1, 0, 0], 20000, 17, None, True)):
        rng = np.random.default_rng(1)
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        x = torch.zeros(sum(lens), K, dtype=torch.bfloat16, device="cuda")
        w, ws = _weights(rng, len(lens), N, K, 0)
        names = kernels_of(lambda: moe.fp8_matmul(x, w, ws, off))
        print("fp8", lens, K, N, names, flush=True)
        assert ("op_fold_kernel" in names) == split
        if tile is None:
            assert "op_f8_stream_kernel" in names and "op_f8_kernel" not in names
        else:
            assert names["op_f8_kernel"][0] == tile and "op_f8_stream_kernel" not in names


@pytest.mark.parametrize("lens,K,N", [([3], 300, 40), ([70, 30], 300, 40), ([700, 900], 144, 2048)])
def test_far_scales(moe, lens, K, N):
    # scales whose products leave fp32's normal range, where the results do not: rows of
    # them beside ordinary ones, streamed and tiled
    rng = np.random.default_rng([K, N])
    M, E, kb = sum(lens), len(lens), -(-K // 128)
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    x, xs = _codes(rng, (M, K)), _scales(rng, (M, kb))
    x[1] = 0x38  # ones
    xs[1] = 2.0**-120
    w, ws = _weights(rng, E, N, K, 0)
    ws = ws * 2.0**-20   # row 1's products: 2^-148 or so each, their sums some 2^-130
    x, xs = x.cuda().view(F8), xs.cuda()
    for scale, back in ((2.0**-120, 1.0), (2.0**-100, 1.0), (2.0**125, 2.0**-26)):
        xs[1] = scale
        y = moe.fp8_matmul(x, w, ws * back, off, x_scale=xs, out_dtype=torch.float32)
        X = _f64(x) * _spread(_f64(xs), M, K, 1)
        W = _f64(w) * _spread(_f64(ws * back), N, K, 128)
        ref, mag = X[1] @ W[0].T, np.abs(X[1]) @ np.abs(W[0].T)
        # (a result below 2^-126 is rounded to 2^-149)
        assert (np.abs(_f64(y)[1] - ref) <= (K + 4) * 2.0**-23 * mag + np.abs(ref) * 2.0**-24 + 2.0**-149).all(), scale
        others = [r for r in range(M) if r != 1]
        e_of = np.repeat(np.arange(E), lens)
        for e in range(E):
            r = [i for i in others if e_of[i] == e]
            ref, mag = X[r] @ W[e].T, np.abs(X[r]) @ np.abs(W[e].T)
            assert (np.abs(_f64(y)[r] - ref) <= (K + 4) * 2.0**-23 * mag + np.abs(ref) * 2.0**-24 + 1e-37).all(), scale


def test_far_scales_of_bf16_results(moe):
    # the same from the 8-bit instruction's tiles, 256 x 256, 128 x 128 and 64 x 64
    rng = np.random.default_rng(17)
    for lens, K, N in (([70, 30], 300, 40), ([700, 900], 144, 2048), ([3000, 5500], 160, 7168)):
        M, kb = sum(lens), -(-K // 128)
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        x, xs = _codes(rng, (M, K)), _scales(rng, (M, kb))
        x[1], xs[1] = 0x38, 2.0**-125  # ones
        w, ws = _weights(rng, len(lens), N, K, 0)
        ws = ws * 2.0**-10
        x, xs = x.cuda().view(F8), xs.cuda()
        y = moe.fp8_matmul(x, w, ws, off, x_scale=xs)
        want = moe.fp8_matmul(x, w, ws, off, x_scale=xs, out_dtype=torch.float32)
        assert torch.equal(y[1], want[1].to(torch.bfloat16)) and (want[1] != 0).any()
        _check_product([2], _f64(y[:2]), x[:2], xs[:2], w[:1], ws[:1], "bf16")


def test_codes_that_are_no_numbers(moe):
    # a NaN code of the rows makes its row NaN, one of the weights its column, no others
    rng = np.random.default_rng(19)
    for lens, K, N in (([3], 300, 40), ([70, 30], 300, 40), ([700, 900], 144, 2048)):
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        x, xs = _codes(rng, (sum(lens), K)), _scales(rng, (sum(lens), -(-K // 128))).cuda()
        w, ws = _weights(rng, len(lens), N, K, 0)
        x[2, K - 1] = 0xFF
        w.view(torch.uint8)[0, 5, 130 % K] = 0x7F
        for odt in ("bf16", "f32"):
            y = moe.fp8_matmul(x.cuda().view(F8), w, ws, off, x_scale=xs, out_dtype=DT[odt])
            bad = torch.isnan(y).cpu()
            want = torch.zeros_like(bad)
            want[2], want[:lens[0], 5] = True, True
            assert torch.equal(bad, want)


def test_many_groups(moe):
    rng = np.random.default_rng(18)
    E, K, N = 700, 136, 24
    lens = [int(v) for v in rng.integers(0, 3, E)]
    M = sum(lens)
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    x, xs = _codes(rng, (M + 9, K)).cuda().view(F8), _scales(rng, (M + 9, 2)).cuda()
    w, ws = _weights(rng, E, N, K, 0)
    y = moe.fp8_matmul(x, w, ws, off, x_scale=xs, out_dtype=torch.float32)
    _check_product(lens, _f64(y), x, xs, w, ws, "f32")
    assert (y[M:] == 0).all()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ties_of_bf16_values(moe, dtype, block_rows):
    # values with bf16's eight bits meet borders exactly, again and again
    rng = np.random.default_rng(20)
    x = torch.from_numpy(rng.standard_normal((3, 256, 512))).to(torch.bfloat16).to(DT[dtype]).cuda()
    x[1] = (x[1].float() * 2.0**-110).to(DT[dtype])
    x[2] = (x[2].float() * 2.0**110).to(DT[dtype])
    q, s = moe.quantize_fp8(x, block_rows=block_rows)
    _check_codes(_f64(x), q, s, block_rows, "ties")


def test_not_finite(moe):
    # a block that holds an infinity or a NaN makes its row NaN and no other; zero blocks
    # and rows of zeros give zeros
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((270, 300))).to(torch.bfloat16).cuda()
    w, ws = moe.quantize_fp8(torch.from_numpy(rng.standard_normal((2, 80, 300)).astype(np.float32)).cuda(), block_rows=128)
    for lens in ([130, 140], [2, 3]):
        M = sum(lens)
        off = torch.tensor([0, lens[0], M], dtype=torch.int32, device="cuda")
        v = x[:M].clone()
        v[1, 9], v[M - 1, 299], v[2] = float("nan"), float("-inf"), 0
        y = moe.fp8_matmul(v, w, ws, off)
        assert torch.isnan(y[1]).all() and torch.isnan(y[M - 1]).all() and (y[2] == 0).all()
        rest = [r for r in range(M) if r not in (1, M - 1)]
        assert torch.isfinite(y[rest]).all()


def test_gradient_of_x(moe):
    # dx = dy W by the same call on the transposed codes, odd sizes among them; against
    # the float64 product of what the codes stand for, and differences of y
    rng = np.random.default_rng(12)
    lens, K, N = [70, 0, 33], 200, 300
    off = torch.tensor([0, 70, 70, 103], dtype=torch.int32, device="cuda")
    w, ws = _weights(rng, 3, N, K, 0)
    dy = torch.from_numpy(rng.standard_normal((103, N))).float().cuda()
    wt, wst = w.view(torch.uint8).transpose(1, 2).contiguous().view(F8), ws.transpose(1, 2).contiguous()
    dx = moe.fp8_matmul(dy, wt, wst, off, out_dtype=torch.float32)
    q, s = moe.quantize_fp8(dy)
    _check_product(lens, _f64(dx), q, s, wt, wst, "f32")
    # the loss <dy, y(x)>: linear in x, so a step of one element changes it by dx there, up
    # to the codes of dy: 2^-4 of each of its products
    W = _f64(w) * _spread(_f64(ws), N, K, 128)
    D = _f64(dy)
    for r, c in ((0, 0), (69, 199), (80, 5), (102, 128)):
        e = 0 if r < 70 else 2
        diff = D[r] @ W[e][:, c]
        assert abs(diff - _f64(dx)[r, c]) <= 2.0**-4 * (np.abs(D[r]) @ np.abs(W[e][:, c]))


def test_offsets_and_defaults(moe):
    rng = np.random.default_rng(10)
    x = torch.from_numpy(rng.standard_normal((40, 64))).to(torch.bfloat16).cuda()
    w, ws = _weights(rng, 3, 64, 64, 0)
    offs = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    good = moe.fp8_matmul(x, w, ws, offs(0, 16, 40, 40))
    assert torch.equal(moe.fp8_matmul(x, w, ws, offs(-5, 16, 1000, 2000)), good)
    y = moe.fp8_matmul(x, w[0], ws[0])
    assert y.dtype == torch.bfloat16 and torch.equal(y[:16], good[:16])
    y = moe.fp8_matmul(x, w[:1], ws[:1], offs(10, 30), out_dtype=torch.float32)
    assert (y[:10] == 0).all() and (y[30:] == 0).all() and (y[10:30] != 0).any()
    assert moe.fp8_matmul(x[:0], w, ws, offs(0, 0, 0, 0)).shape == (0, 64)


def test_streams_and_graph_replay(moe):
    rng = np.random.default_rng(11)
    jobs = []
    for lens, K, N in (([40, 0, 100, 77], 264, 136), ([40, 30], 20000, 33), ([1, 0, 2], 4096, 130), ([700, 900], 144, 2048)):
        off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        jobs.append((torch.from_numpy(rng.standard_normal((sum(lens), K))).to(torch.bfloat16).cuda(),
                     *_weights(rng, len(lens), N, K, 0), off))

    def run(xs):
        out = []
        for x, (_, w, ws, off) in zip(xs, jobs):
            q, s = moe.quantize_fp8(x)
            out += [moe.fp8_matmul(x, w, ws, off), moe.fp8_matmul(q, w, ws, off, x_scale=s, out_dtype=torch.float32), s]
        return out

    first = [j[0] for j in jobs]
    sets = [first, [x * 3 for x in first], [x * -0.3 for x in first]]
    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(((turn + k) % 3, run(sets[(turn + k) % 3])))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, res in got for a, b in zip(res, want[i]))
    bufs = [[x.clone() for x in first] for _ in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(b))
        graphs.append(g)
    for i, k in ((0, 1), (1, 2), (2, 0), (1, 1)):
        for b, n in zip(bufs, (i, k)):
            for x, v in zip(b, sets[n]):
                x.copy_(v)
        streams[0].wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(streams[0]):
            graphs[1].replay()
        eager = run(sets[k])
        torch.cuda.synchronize()
        for res, n in ((outs[0], i), (outs[1], k), (eager, k)):
            assert all(torch.equal(a, b) for a, b in zip(res, want[n])), (i, k)


def test_written_results_are_seen_by_autograd(moe):
    rng = np.random.default_rng(2)
    w, ws = _weights(rng, 1, 6, 8, 0)
    out = torch.zeros(4, 6, device="cuda")
    before = out._version
    moe.fp8_matmul(torch.randn(4, 8, device="cuda"), w, ws, out=out)
    assert out._version > before


def test_weights_past_2_31_elements(moe):
    # a matrix whose rows start past 2^31 elements: rows far apart in a large buffer
    rng = np.random.default_rng(4)
    N, K, ld = 600, 256, (1 << 22) + 48
    buf = torch.zeros(N * ld, dtype=torch.uint8, device="cuda")
    w = buf.as_strided((1, N, K), (N * ld, ld, 1))
    w.copy_(_codes(rng, (1, N, K)).cuda())
    ws = _scales(rng, (1, 5, 2)).cuda()
    for M in (3, 200):
        x, xs = _codes(rng, (M, K)).cuda().view(F8), _scales(rng, (M, 2)).cuda()
        y = moe.fp8_matmul(x, w.view(F8), ws, x_scale=xs, out_dtype=torch.float32)
        _check_product([M], _f64(y), x, xs, w.contiguous().view(F8), ws, "f32")


def test_gated_block_served_in_8_bits(moe):
    # the operators together, as a server uses them: gated projections in bf16, their
    # result quantised in the call, the down product in 8 bits
    rng = np.random.default_rng(15)
    lens, K, H, N = [33, 0, 70], 96, 260, 80
    off = torch.tensor([0, 33, 33, 103], dtype=torch.int32, device="cuda")
    new = lambda *s, by=1.0: torch.from_numpy(rng.standard_normal(s) * by).to(torch.bfloat16).cuda()
    x, w1, w3 = new(103, K), new(3, H, K, by=K**-0.5), new(3, H, K, by=K**-0.5)
    w2, w2s = moe.quantize_fp8(new(3, N, H, by=H**-0.5), block_rows=128)
    h = moe.gated_matmul(x, w1, w3, off)
    y = moe.fp8_matmul(h, w2, w2s, off, out_dtype=torch.float32)
    q, s = moe.quantize_fp8(h)
    _check_product(lens, _f64(y), q, s, w2, w2s, "f32")
