"""fp8_matmul with scales far from one, in every form: a row's results depend on its own
scales and its groups' weights alone, to the bit, and are the float64 formula's wherever
fp32 holds them.  Tolerances: test_gpu_ops_fp8.py's (_check_product), with 2^-149, fp32's
last place, in place of its absolute term."""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = {"bf16": 2.0**-8, "f32": 2.0**-24}
# streamed; 64, 128 and 256 (bf16 result) rows in a tile; k split over tiles
SHAPES = [([3, 4], 520, 300), ([70, 30], 520, 300), ([700, 900], 400, 2048), ([3000, 5500], 400, 7168), ([40, 30], 20000, 33)]


def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _codes(rng, shape):
    return torch.from_numpy((rng.integers(0, 127, shape) | (rng.integers(0, 2, shape) << 7)).astype(np.uint8))


def _inputs(rng, lens, K, N):
    M, E, kb = sum(lens), len(lens), -(-K // 128)
    scales = lambda *s: torch.from_numpy(rng.uniform(0.001, 0.02, s).astype(np.float32)).cuda()
    return (_codes(rng, (M, K)).cuda(), scales(M, kb), _codes(rng, (E, N, K)).cuda(), scales(E, -(-N // 128), kb),
            _offsets(lens))


def _run(moe, x, xs, w, ws, off, odt):
    return moe.fp8_matmul(x.view(F8), w.view(F8), ws, off, x_scale=xs, out_dtype=DT[odt])


def _row(x, xs, w, ws, r, e):
    """Row r's results by weight e in float64, and the sums of their magnitudes."""
    K, N = w.shape[2], w.shape[1]
    X = x[r].view(F8).double() * xs[r].double().repeat_interleave(128)[:K]
    W = w[e].view(F8).double() * ws[e].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (W * X).sum(1), (W * X).abs().sum(1)


def _near(y, ref, mag, K, odt, what, cut=True):
    tol = (K + 4) * 2.0**-23 * mag + ref.abs() * STEP[odt] + 2.0**-149
    if odt == "bf16":
        tol = tol + (7 * 2.0**-13 if cut else 0) * mag + 2.0**-134  # (bf16's last place)
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()))


@pytest.mark.parametrize("odt", ["f32", "bf16"])
@pytest.mark.parametrize("lens,K,N", SHAPES)
def test_one_far_block_leaves_the_other_results_alone(moe, lens, K, N, odt):
    rng = np.random.default_rng([K, N, 1])
    x, xs, w, ws, off = _inputs(rng, lens, K, N)
    want, M = _run(moe, x, xs, w, ws, off, odt), sum(lens)
    print(lens, K, N, odt, kernels_of(lambda: _run(moe, x, xs, w, ws, off, odt)), flush=True)
    others = torch.arange(M, device="cuda") != 2
    for far in (1e-36, 1e-44, 2.0**60, 2.0**90):  # a block of row 2
        s = xs.clone()
        s[2, 3] = far
        y = _run(moe, x, s, w, ws, off, odt)
        assert torch.equal(y[others], want[others]), far
        _near(y[2], *_row(x, s, w, ws, 2, 0), K, odt, far)
    kept = torch.ones_like(want, dtype=torch.bool)
    kept[:lens[0], :128] = False
    for far in (1e-36, 1e-44, 2.0**60):  # a block of the first group's weight
        s = ws.clone()
        s[0, 0, 3] = far
        y = _run(moe, x, xs, w, s, off, odt)
        assert torch.equal(y[kept], want[kept]), far
        for r in (0, 1, lens[0] - 1):
            _near(y[r], *_row(x, xs, w, s, r, 0), K, odt, far)


@pytest.mark.parametrize("odt", ["f32", "bf16"])
@pytest.mark.parametrize("lens,K,N", SHAPES)
def test_small_products_beside_large_scales(moe, lens, K, N, odt):
    # all codes of the blocks with ordinary scales are zero: the sum is that of one block
    # whose scale product is far below fp32's normal range
    rng = np.random.default_rng([K, N, 2])
    x, xs, w, ws, off = _inputs(rng, lens, K, N)
    x[1, :128] = x[1, 256:] = 0
    xs[1, 1] = 2.0**-118
    w[0, :, 128:256] = 0x38  # ones: products that the 8-bit instruction sums as they are
    x[1, 128:256] = 0x38
    y = _run(moe, x, xs, w, ws, off, odt)[1]
    ref, mag = _row(x, xs, w, ws, 1, 0)
    assert (ref < 2.0**-116).all() and (ref > 2.0**-126).all()
    _near(y, ref, mag, K, odt, "small", cut=False)


@pytest.mark.parametrize("lens,K,N", [s for s in SHAPES if s[1] < 20000])
def test_large_sums_that_cancel(moe, lens, K, N):
    # blocks of 2^131 and -2^131 leave a sum that fp32 holds: finite, whatever the form
    M, E, kb = sum(lens), len(lens), -(-K // 128)
    x = torch.zeros(M, K, dtype=torch.uint8, device="cuda")
    w = torch.zeros(E, N, K, dtype=torch.uint8, device="cuda")
    x[:, :128], x[:, 128:256], w[:, :, :256] = 0x38, 0xB8, 0x38  # 128 ones, 128 minus ones
    w[:, :, 255] = 0x34                                          # 0.75
    xs, ws = torch.full((M, kb), 2.0**70, device="cuda"), torch.full((E, -(-N // 128), kb), 2.0**54, device="cuda")
    for odt in ("f32", "bf16"):
        y = _run(moe, x, xs, w, ws, _offsets(lens), odt)
        assert (y == 2.0**122).all(), (odt, y.flatten()[:3].tolist())


def test_split_sums_that_fp32_holds(moe):
    # the ranges' sums of a split k are in fp32: far products that stay inside it
    K, N, M = 20000, 33, 70
    x, w = torch.full((M, K), 0x38, dtype=torch.uint8, device="cuda"), torch.full((1, N, K), 0x38, dtype=torch.uint8, device="cuda")
    kb = -(-K // 128)
    for a, b in ((2.0**60, 2.0**50), (2.0**-70, 2.0**-60), (2.0**-149, 2.0**20)):
        xs, ws = torch.full((M, kb), a, device="cuda"), torch.full((1, 1, kb), b, device="cuda")
        y = _run(moe, x, xs, w, ws, None, "f32")
        assert (y.double() == K * a * b).all(), (a, b)


@pytest.mark.parametrize("odt", ["f32", "bf16"])
@pytest.mark.parametrize("lens,K,N", SHAPES)
def test_scales_that_are_no_numbers(moe, lens, K, N, odt):
    # a NaN or an infinity, alone and beside a far one, leaves no finite number in its row and
    # every other row as it was; one of a weight in its group's columns
    rng = np.random.default_rng([K, N, 3])
    x, xs, w, ws, off = _inputs(rng, lens, K, N)
    x[2] = 0x38  # ones, so that no sum is 0
    w[0, :, 128:256] = 0x30
    want, M = _run(moe, x, xs, w, ws, off, odt), sum(lens)
    others = torch.arange(M, device="cuda") != 2
    for bad, beside in ((float("nan"), 0.01), (float("inf"), 0.01), (float("nan"), 2.0**90), (float("nan"), 1e-40)):
        s = xs.clone()
        s[2, 1], s[2, 0] = bad, beside
        y = _run(moe, x, s, w, ws, off, odt)
        assert torch.equal(y[others], want[others]) and not torch.isfinite(y[2]).any(), (bad, beside)
        assert torch.isnan(y[2]).all() or bad == float("inf")
    s = ws.clone()
    s[0, 0, 1] = float("nan")
    y = _run(moe, x, xs, w, s, off, odt)
    assert torch.isnan(y[:lens[0], :128]).all()
    assert torch.equal(y[:, 128:], want[:, 128:]) and torch.equal(y[lens[0]:], want[lens[0]:])
