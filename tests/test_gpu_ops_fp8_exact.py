"""fp8_matmul where its products have to be exact: with ``exact``, and without it on the
way to a bfloat16 result of few rows and of sums whose k was split.  The sums of such a
call are those of the float32 result, so the bfloat16 one is that, rounded once: the
same bits.  (The float32 result against float64: test_gpu_ops_fp8.py.)"""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _codes(rng, shape):
    """Any finite codes."""
    return torch.from_numpy((rng.integers(0, 127, shape) | (rng.integers(0, 2, shape) << 7)).astype(np.uint8))


def _scales(rng, shape):
    return torch.from_numpy(rng.uniform(0.001, 0.02, shape).astype(np.float32)).cuda()


def _inputs(rng, lens, K, N, xt, pad):
    M, E = sum(lens), len(lens)
    t = torch.full((E, N, K + pad), 0x7F, dtype=torch.uint8)  # NaN behind the rows
    t[:, :, :K] = _codes(rng, (E, N, K))
    w, ws = t.cuda().view(F8)[:, :, :K], _scales(rng, (E, -(-N // 128), -(-K // 128)))
    if xt == "codes":
        return _codes(rng, (M, K)).cuda().view(F8), w, ws, dict(x_scale=_scales(rng, (M, -(-K // 128))))
    return torch.from_numpy(rng.standard_normal((M, K))).to(DT[xt]).cuda(), w, ws, {}


# group lengths, K, N: one row, streamed, 64, 128 and 256-row tiles (256: without ``exact``
# alone), odd sizes, k split over tiles and over streams
SHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([2], 4096, 130),
    ([33, 130, 5, 0, 300], 208, 136),
    ([16, 16, 40, 2], 129, 257),
    ([700, 0, 900, 500], 144, 2048),
    ([3000, 5500], 160, 7168),
    ([40, 30], 20000, 33),
    ([0, 9, 0], 5001, 50),
    ([0, 0, 2, 0, 1, 0, 0], 20000, 17),
]


@pytest.mark.parametrize("pad", [0, 12, 5])
@pytest.mark.parametrize("xt", ["bf16", "f32", "codes"])
def test_exact(moe, xt, pad):
    for lens, K, N in SHAPES:
        print(f"exact fp8 {xt} pad={pad} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, pad, 6])
        x, w, ws, kw = _inputs(rng, lens, K, N, xt, pad)
        off, res = _offsets(lens), []
        names = kernels_of(lambda: res.append(moe.fp8_matmul(x, w, ws, off, exact=True, **kw)))
        assert "op_f8_stream_kernel" in names or names["op_f8_kernel"][7] == "true"  # the codes in bf16
        y = moe.fp8_matmul(x, w, ws, off, out_dtype=torch.float32, **kw)
        assert res[0].dtype == torch.bfloat16 and torch.equal(res[0], y.to(torch.bfloat16))
        assert torch.equal(moe.fp8_matmul(x, w, ws, off, out_dtype=torch.float32, exact=True, **kw), y)


@pytest.mark.parametrize("xt", ["bf16", "f32", "codes"])
def test_few_rows_and_split_sums_are_exact_by_themselves(moe, xt):
    for lens, K, N, kernel in (([1], 1, 1, "stream"), ([0, 3, 0], 7, 5, "stream"), ([2], 4096, 130, "stream"),
                               ([40, 30], 20000, 33, "split"), ([0, 9, 0], 5001, 50, "split"),
                               ([0, 0, 2, 0, 1, 0, 0], 20000, 17, "stream")):
        print(f"fp8 {xt}->bf16 lens={lens} K={K} N={N}", flush=True)
        x, w, ws, kw = _inputs(np.random.default_rng([K, N, 7]), lens, K, N, xt, 0)
        off, res = _offsets(lens), []
        names = kernels_of(lambda: res.append(moe.fp8_matmul(x, w, ws, off, **kw)))
        assert ("op_f8_stream_kernel" in names) if kernel == "stream" else names["op_f8_kernel"][7] == "true"
        assert torch.equal(res[0], moe.fp8_matmul(x, w, ws, off, out_dtype=torch.float32, **kw).to(torch.bfloat16))


def test_a_small_product_beside_a_large_one(moe):
    # 16 * 16, cancelling, beside 2^-16 of it in every eight codes: the sum is the small
    # products', and every partial sum is a multiple of 2^-8 below 2^13, so fp32 holds it
    K, N, M = 256, 160, 200
    x, w = torch.zeros(M, K, dtype=torch.uint8), torch.zeros(1, N, K, dtype=torch.uint8)
    x[:, 0::8], w[:, :, 0::8] = 0x58, 0x58  # 16
    w[:, :, 8::16] = 0xD8                   # -16
    x[:, 1::8], w[:, :, 1::8] = 0x18, 0x18  # 2^-4
    x, w = x.cuda().view(F8), w.cuda().view(F8)
    xs, ws = torch.ones(M, 2, device="cuda"), torch.ones(1, 2, 2, device="cuda")
    y = moe.fp8_matmul(x, w, ws, x_scale=xs, exact=True)
    assert (y == 32 * 2.0**-8).all()
