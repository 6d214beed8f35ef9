"""Long sums of the gated and the 8-bit products, held so near that one product lost or
counted twice shows.

A sum of K products p with independent signs: every partial sum has the standard
deviation t = sqrt(sum p^2) at most, each of its K roundings (and of fp32 operands'
products') is at most 2^-24 of it, of either sign: sqrt(K) 2^-24 t, and eight times that
for the furthest of all elements.  A lost product is t / sqrt(K) on average: 10^3 times
as much at K = 16401."""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FLUX, LLAMA = 0, 1
F8 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
# group lengths, K, N: k split over streams and tiles, and whole; ends inside ranges
LONG = [([1], 8192, 16), ([3, 0, 2], 4001, 125), ([3, 0, 2], 16401, 45), ([71], 5440, 64), ([200, 0, 150], 3456, 131),
        ([40, 3], 2999, 64), ([40, 30], 20000, 33), ([600, 500], 4100, 1040)]


def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _near(y, terms, K, step, what):
    """terms: pairs of matrices (rows, k), (k, columns) whose products are summed."""
    ref = sum(a @ b for a, b in terms)
    t = sum((a * a) @ (b * b) for a, b in terms).sqrt()
    tol = 8 * K**0.5 * 2.0**-24 * t + ref.abs() * step
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), ((y.double() - ref).abs() / tol).max().item())


def _groups(lens):
    at = 0
    for e, n in enumerate(lens):
        if n:
            yield e, slice(at, at + n)
        at += n


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_gated(moe, dtype, odt, layout):
    step = {"bf16": 2.0**-8, "f32": 2.0**-24}
    for lens, K, N in LONG:
        g = torch.Generator(device="cuda").manual_seed(K + N)
        E, M, off = len(lens), sum(lens), _offsets(lens)
        new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[dtype])
        mat = lambda: new(E, N, K) if layout == LLAMA else new(E, K, N)
        out_in = lambda w, e: (w[e] if layout == LLAMA else w[e].t()).double().contiguous()
        x, w1, w3 = new(M, K), mat(), mat()
        kw = dict(activation=moe.identity, layout=layout)
        print(f"long gated {dtype}->{odt} layout={layout} lens={lens} K={K} N={N}", flush=True)
        h, a, b = moe.gated_matmul(x, w1, w3, off, out_dtype=DT[odt], save=True, **kw)
        w2 = new(E, K, N) if layout == LLAMA else new(E, N, K)  # out_dim K
        one = torch.ones(M, N, device="cuda", dtype=DT[dtype])
        da, db, h2 = moe.gated_matmul_grad(x, one, one, w2, off, **kw)  # dh, twice
        # (the hidden size is the long one)
        v1, v3 = (new(E, K, N) if layout == LLAMA else new(E, N, K) for _ in range(2))
        d1, d3 = new(M, K), new(M, K)
        dx = moe.gated_matmul_grad_x(d1, d3, v1, v3, off, layout=layout, out_dtype=DT[odt])
        for e, s in _groups(lens):
            X, wa, wb = x[s].double(), out_in(w1, e).t(), out_in(w3, e).t()
            _near(a[s], [(X, wa)], K, step[dtype], "a")
            _near(b[s], [(X, wb)], K, step[dtype], "b")
            ra, rb = X @ wa, X @ wb
            ta, tb = ((X * X) @ (w * w) for w in (wa, wb))
            d = 8 * K**0.5 * 2.0**-24  # of t: a b is off by a's part times b and b's times a
            tol = d * (ta.sqrt() * rb.abs() + tb.sqrt() * ra.abs()) * 1.001 + (ra * rb).abs() * (step[odt] + 2.0**-24) + d * d * (ta * tb).sqrt()
            assert ((h[s].double() - ra * rb).abs() <= tol).all(), "h"
            W2 = out_in(w2, e)  # (K, N)
            _near(da[s], [(X, W2)], K, step[dtype], "da")
            _near(db[s], [(X, W2)], K, step[dtype], "db")
            _near(dx[s], [(d1[s].double(), out_in(v1, e)), (d3[s].double(), out_in(v3, e))], 2 * K, step[odt], "dx")
        assert (h2[:M] == 1).all()


@pytest.mark.parametrize("odt", ["f32", "bf16"])
def test_fp8(moe, odt):
    # codes of all magnitudes, exact products: a block's sum and the sum of blocks
    for lens, K, N in LONG:
        rng = np.random.default_rng([K, N, 3])
        E, M, kb, off = len(lens), sum(lens), -(-K // 128), _offsets(lens)
        codes = lambda *s: torch.from_numpy((rng.integers(0, 127, s) | (rng.integers(0, 2, s) << 7)).astype(np.uint8)).cuda().view(F8)
        scales = lambda *s: torch.from_numpy(rng.uniform(0.001, 0.02, s).astype(np.float32)).cuda()
        x, xs, w, ws = codes(M, K), scales(M, kb), codes(E, N, K), scales(E, -(-N // 128), kb)
        names = kernels_of(lambda: moe.fp8_matmul(x, w, ws, off, x_scale=xs, exact=True))
        print(f"long fp8 {odt} lens={lens} K={K} N={N} {sorted(names)}", flush=True)
        y = moe.fp8_matmul(x, w, ws, off, x_scale=xs, out_dtype=DT[odt], exact=True)
        for e, s in _groups(lens):
            X = x[s].double() * xs[s].double().repeat_interleave(128, 1)[:, :K]
            W = w[e].double() * ws[e].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
            # (and the product of the two scales and its own with a block's sum: 2^-23 of both)
            _near(y[s], [(X, W.t().contiguous())], K + 16, {"bf16": 2.0**-8, "f32": 2.0**-24}[odt], "y")
