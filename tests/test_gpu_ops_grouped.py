"""The grouped products and their gradients (grouped_matmul*, ops.py) against
float64 products of the same inputs.

Tolerance per element: K products summed in fp32 are off by at most K * 2^-23
of the sum of their magnitudes (every addition rounds by at most one fp32 step,
whatever the order or the rounding mode of the matrix unit), then one rounding
to the result's type, at most half a step (2^-8 of a bf16 value, 2^-24 of an
fp32 one)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FLUX, LLAMA = 0, 1
SENTINEL = 776.0  # exact in bf16 and fp32
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rows(rng, rows, cols, dtype, pad, tail=0):
    """rows + tail rows of a wider tensor; the padding columns and the rows
    past the groups hold NaN."""
    t = torch.full((rows + tail, cols + pad), float("nan"), dtype=DT[dtype])
    t[:rows, :cols] = torch.from_numpy(rng.standard_normal((rows, cols))).to(DT[dtype])
    return t.cuda()[:, :cols]


def _mats(rng, E, a, b, dtype, pad):
    t = torch.full((E, a, b + pad), float("nan"), dtype=DT[dtype])
    t[:, :, :b] = torch.from_numpy(rng.standard_normal((E, a, b))).to(DT[dtype])
    return t.cuda()[:, :, :b]


def _f64(t):
    return t.detach().cpu().double().numpy()


def _close(got, ref, mag, K, dtype):
    tol = K * 2.0**-23 * mag + np.abs(ref) * {"bf16": 2.0**-8, "f32": 2.0**-24}[dtype] + 1e-35
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - ref).max()))


def _offsets(lens, start=0):
    return torch.tensor(np.concatenate([[start], start + np.cumsum(lens)]), dtype=torch.int32, device="cuda")


# group lengths, K, N: no rows, one row, odd sizes below, at and past the tiles' edges
SHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([17, 0, 1, 64], 64, 96),
    ([33, 130, 5, 0, 300], 200, 136),
    ([16, 16, 31, 2], 129, 257),
    ([70, 90, 65], 333, 72),
    ([0, 0], 40, 24),
    ([5] * 70, 96, 48),            # more groups than a wave has lanes
    ([700, 0, 900, 500], 72, 2048),  # 128 x 128 tiles
]


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_rows_products(moe, dtype, odt, layout, pad):
    for lens, K, N in SHAPES:
        print(f"grouped rows {dtype}->{odt} layout={layout} pad={pad} lens={lens[:6]} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, pad])
        M, E, tail = sum(lens), len(lens), 5
        off = _offsets(lens)
        shape = (N, K) if layout == LLAMA else (K, N)
        w = _mats(rng, E, *shape, dtype, pad)
        W = _f64(w) if layout == LLAMA else _f64(w).transpose(0, 2, 1)
        for grad in (False, True):
            src = _rows(rng, M, N if grad else K, dtype, pad, tail)
            out = torch.full((M + tail, (K if grad else N) + pad), SENTINEL, dtype=DT[odt], device="cuda")
            view = out[:, :K if grad else N]
            fn = moe.grouped_matmul_grad_x if grad else moe.grouped_matmul
            assert fn(src, w, off, layout=layout, out=view) is view
            got, s, at = _f64(view), _f64(src), 0
            for e, n in enumerate(lens):
                m = W[e] if grad else W[e].T
                a = s[at:at + n]
                _close(got[at:at + n], a @ m, np.abs(a) @ np.abs(m), N if grad else K, odt)
                at += n
            # rows past the groups and columns past the rows stay as they were
            assert (got[M:] == SENTINEL).all() and (_f64(out)[:, view.shape[1]:] == SENTINEL).all()


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_large_tiles(moe, layout):
    # 256 x 256 tiles (both operand orders), ragged last tiles, K with a part stage
    rng = np.random.default_rng(5)
    lens, K, N = [2100, 1, 3000, 3400], 136, 4040
    print(f"grouped 256-row tiles layout={layout}", flush=True)
    shape = (N, K) if layout == LLAMA else (K, N)
    w, x = _mats(rng, 4, *shape, "bf16", 0), _rows(rng, sum(lens), K, "bf16", 0)
    y = moe.grouped_matmul(x, w, _offsets(lens), layout=layout)
    dy = _rows(rng, sum(lens), N, "bf16", 0)
    dx = moe.grouped_matmul_grad_x(dy, w, _offsets(lens), layout=layout)
    W, X, D, at = _f64(w), _f64(x), _f64(dy), 0
    for e, n in enumerate(lens):
        m = W[e].T if layout == LLAMA else W[e]  # (K, N)
        s = slice(at, at + n)
        _close(_f64(y[s]), X[s] @ m, np.abs(X[s]) @ np.abs(m), K, "bf16")
        _close(_f64(dx[s]), D[s] @ m.T, np.abs(D[s]) @ np.abs(m.T), N, "bf16")
        at += n


# long sums for few rows and columns: k split over workgroups, streamed and
# tiled, whole and odd lengths
LONG = [([1], 8192, 16), ([3, 0, 2], 4001, 125), ([3, 0, 2], 16401, 125), ([71], 5440, 64), ([200, 0, 150], 3456, 131), ([40, 3], 2999, 64)]


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_long_sums(moe, dtype, odt, layout):
    for lens, K, N in LONG:
        print(f"grouped long sum {dtype}->{odt} layout={layout} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, 2])
        M, E, start = sum(lens), len(lens), 2
        x = _rows(rng, M + start, K, dtype, 0, 4)
        w = _mats(rng, E, *((N, K) if layout == LLAMA else (K, N)), dtype, 0)
        W, X = (_f64(w) if layout == LLAMA else _f64(w).transpose(0, 2, 1)), _f64(x)
        out = torch.full((M + start + 4, N + 3), SENTINEL, dtype=DT[odt], device="cuda")
        y = moe.grouped_matmul(x, w, _offsets(lens, start), layout=layout, out=out[:, :N])
        got, at = _f64(y), start
        for e, n in enumerate(lens):
            a = X[at:at + n]
            _close(got[at:at + n], a @ W[e].T, np.abs(a) @ np.abs(W[e].T), K, odt)
            at += n
        assert (got[:start] == SENTINEL).all() and (got[at:] == SENTINEL).all() and (_f64(out)[:, N:] == SENTINEL).all()


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_large_weight_gradient_tiles(moe, layout):
    # 256 x 256 tiles: groups whose matrices fill the GPU by themselves
    rng = np.random.default_rng(6)
    lens, K, N = [70, 0, 133], 4096, 2040
    x, dy = _rows(rng, 203, K, "bf16", 0), _rows(rng, 203, N, "bf16", 0)
    dw = moe.grouped_matmul_grad_w(x, dy, _offsets(lens), layout=layout, out_dtype=torch.float32)
    a, b = (_f64(dy), _f64(x)) if layout == LLAMA else (_f64(x), _f64(dy))
    for e, s in enumerate((slice(0, 70), slice(70, 70), slice(70, 203))):
        _close(_f64(dw[e]), a[s].T @ b[s], np.abs(a[s]).T @ np.abs(b[s]), max(lens[e], 1), "f32")


WSHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([17, 0, 1, 64], 64, 96),
    ([33, 130, 5, 0, 300], 200, 136),
    ([129, 65, 0], 333, 71),
    ([100, 40, 0, 64], 1024, 1024),           # 128 x 128 tiles
    ([70, 0, 64, 1, 200, 66, 2, 30], 2048, 2040),  # 256 x 256 tiles
    ([3000], 96, 40),                          # a long sum for few tiles
    ([2500, 0, 4000], 64, 64),
]


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_weight_gradient(moe, dtype, odt, layout, pad):
    for lens, K, N in WSHAPES:
        print(f"grad_w {dtype}->{odt} layout={layout} pad={pad} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, pad, 1])
        M, E, tail = sum(lens), len(lens), 3
        x, dy = _rows(rng, M, K, dtype, pad, tail), _rows(rng, M, N, dtype, pad, tail)
        off = _offsets(lens)
        shape = (N, K) if layout == LLAMA else (K, N)
        buf = torch.full((E, shape[0], shape[1] + pad), SENTINEL, dtype=DT[odt], device="cuda")
        out = buf[:, :, :shape[1]]
        moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out=out)
        a, b = (_f64(dy), _f64(x)) if layout == LLAMA else (_f64(x), _f64(dy))
        got, at = _f64(out), 0
        refs = []
        for e, n in enumerate(lens):
            s = slice(at, at + n)
            ref, mag = a[s].T @ b[s], np.abs(a[s]).T @ np.abs(b[s])
            refs.append((ref, mag))
            _close(got[e], ref, mag, max(n, 1), odt)
            at += n
        assert (_f64(buf)[:, :, shape[1]:] == SENTINEL).all()
        # accumulate: what out held, plus the sums (one more fp32 addition)
        base = torch.from_numpy(rng.standard_normal((E, *shape))).to(DT[odt]).cuda()
        acc = base.clone()
        moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out=acc, accumulate=True)
        for e, (ref, mag) in enumerate(refs):
            p = _f64(base)[e]
            _close(_f64(acc)[e], ref + p, mag + np.abs(p), max(lens[e], 1) + 1, odt)


def test_one_expert_and_defaults(moe):
    rng = np.random.default_rng(8)
    x, w, dy = _rows(rng, 50, 24, "bf16", 0), _mats(rng, 1, 40, 24, "bf16", 0), _rows(rng, 50, 40, "bf16", 0)
    y = moe.grouped_matmul(x, w[0], out_dtype=torch.float32)
    assert y.dtype == torch.float32 and y.shape == (50, 40)
    X, W, D = _f64(x), _f64(w[0]), _f64(dy)
    _close(_f64(y), X @ W.T, np.abs(X) @ np.abs(W.T), 24, "f32")
    dw = moe.grouped_matmul_grad_w(x, dy)
    assert dw.shape == (40, 24) and dw.dtype == torch.bfloat16
    _close(_f64(dw), D.T @ X, np.abs(D.T) @ np.abs(X), 50, "bf16")
    # rows outside every group, when the call makes the result: zeros
    off = torch.tensor([10, 30], dtype=torch.int32, device="cuda")
    y = moe.grouped_matmul(x, w, off)
    assert (y[:10] == 0).all() and (y[30:] == 0).all() and (y[10:30] != 0).any()
    # no rows at all
    assert moe.grouped_matmul(x[:0], w, _offsets([0])).shape == (0, 40)
    assert (moe.grouped_matmul_grad_w(x[:0], dy[:0], _offsets([0, 0])) == 0).all()


def test_infinities_stay_in_their_rows(moe):
    rng = np.random.default_rng(9)
    x, w = _rows(rng, 200, 72, "bf16", 0), _mats(rng, 2, 72, 72, "bf16", 0)
    x[5, 3], x[150, 71] = float("inf"), float("nan")
    y = moe.grouped_matmul(x, w, _offsets([100, 100]))
    fin = torch.isfinite(y).all(dim=1).cpu()
    assert not fin[5] and not fin[150] and fin.sum() == 198


def test_offsets_out_of_range_stay_in_bounds(moe):
    # offsets past the rows are held within them: group 1 gets the rest, group 2 nothing
    rng = np.random.default_rng(10)
    x, w = _rows(rng, 40, 64, "bf16", 0), _mats(rng, 3, 64, 64, "bf16", 0)
    good = moe.grouped_matmul(x, w, _offsets([16, 24, 0]))
    off = torch.tensor([-5, 16, 1000, 2000], dtype=torch.int32, device="cuda")
    assert torch.equal(moe.grouped_matmul(x, w, off), good)
    dy = _rows(rng, 40, 64, "bf16", 0)
    assert torch.equal(moe.grouped_matmul_grad_w(x, dy, off), moe.grouped_matmul_grad_w(x, dy, _offsets([16, 24, 0])))


def test_streams_and_graph_replay(moe):
    # the same bits on another stream and in every replay of a captured graph,
    # with new inputs copied in between
    rng = np.random.default_rng(11)
    lens = [40, 0, 100, 77]
    off = _offsets(lens)
    xs = [_rows(rng, 217, 264, "bf16", 0) for _ in range(3)]
    dys = [_rows(rng, 217, 136, "bf16", 0) for _ in range(3)]
    w = _mats(rng, 4, 136, 264, "bf16", 0)

    def step(x, dy):
        return (moe.grouped_matmul(x, w, off), moe.grouped_matmul_grad_x(dy, w, off),
                moe.grouped_matmul_grad_w(x, dy, off, out_dtype=torch.float32))

    want = [step(x, dy) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(xs[0], dys[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    x, dy = xs[0].clone(), dys[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, dy)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_wide_strides(moe, dtype):
    # rows 4 MB and more apart: a tile's byte offsets no longer fit the loads'
    # 32 bits, and elements lie past 2^31 from the tensor's start
    print(f"grouped wide strides {dtype}", flush=True)
    rng = np.random.default_rng(12)
    lens, K, N, ld = [150, 0, 100, 170], 136, 72, 2**23 + 8
    M = sum(lens)
    big = torch.empty(M * ld, dtype=DT[dtype], device="cuda")
    assert M * ld > 2**31
    wide = lambda cols: big.as_strided((M, cols), (ld, 1))
    off = _offsets(lens)
    x = _rows(rng, M, K, dtype, 0)
    dy = _rows(rng, M, N, dtype, 0)
    w = {LLAMA: _mats(rng, 4, N, K, dtype, 0)}
    w[FLUX] = w[LLAMA].transpose(1, 2).contiguous()
    for layout in (LLAMA, FLUX):
        y, dx = moe.grouped_matmul(x, w[layout], off, layout=layout), moe.grouped_matmul_grad_x(dy, w[layout], off, layout=layout)
        dw = moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out_dtype=torch.float32)
        X, D = _f64(x), _f64(dy)
        W = _f64(w[LLAMA])
        # operands, then results, in the wide tensor
        xw = wide(K)
        xw.copy_(x)
        got = [moe.grouped_matmul(xw, w[layout], off, layout=layout),
               moe.grouped_matmul_grad_w(xw, dy, off, layout=layout, out_dtype=torch.float32)]
        yw = wide(N)
        moe.grouped_matmul(x, w[layout], off, layout=layout, out=yw)
        got.append(yw.clone())
        yw.copy_(dy)
        got.append(moe.grouped_matmul_grad_x(yw, w[layout], off, layout=layout))
        at = 0
        for e, n in enumerate(lens):
            s = slice(at, at + n)
            for r in (y, got[0], got[2]):
                _close(_f64(r[s]), X[s] @ W[e].T, np.abs(X[s]) @ np.abs(W[e].T), K, dtype)
            for r in (dx, got[3]):
                _close(_f64(r[s]), D[s] @ W[e], np.abs(D[s]) @ np.abs(W[e]), N, dtype)
            g = (D[s].T @ X[s], np.abs(D[s]).T @ np.abs(X[s]))
            if layout == FLUX:
                g = tuple(m.T for m in g)
            for r in (dw, got[1]):
                _close(_f64(r[e]), *g, max(n, 1), "f32")
            at += n


@pytest.mark.parametrize("pad", [0, 2, 6])
@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_rows_of_whole_dwords(moe, layout, pad):
    # bf16 rows of an even length that do not start on 16 bytes: loaded by chunks
    # whose last one may reach into the next row (or its padding, NaN here)
    for lens, K, N in (([1, 0, 30], 2, 6), ([3, 40], 18, 22), ([33, 130, 5, 0, 300], 202, 134), ([700, 0, 900, 500], 70, 2046),
                       ([100, 40, 0, 64], 1022, 1026), ([71], 5442, 62)):
        print(f"grouped dword rows layout={layout} pad={pad} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, pad, 4])
        M, E = sum(lens), len(lens)
        w = _mats(rng, E, *((N, K) if layout == LLAMA else (K, N)), "bf16", pad)
        x, dy, off = _rows(rng, M, K, "bf16", pad), _rows(rng, M, N, "bf16", pad), _offsets(lens)
        y, dx = moe.grouped_matmul(x, w, off, layout=layout), moe.grouped_matmul_grad_x(dy, w, off, layout=layout)
        dw = _f64(moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out_dtype=torch.float32))
        W = _f64(w) if layout == LLAMA else _f64(w).transpose(0, 2, 1)
        X, D, Y, DX, at = _f64(x), _f64(dy), _f64(y), _f64(dx), 0
        for e, n in enumerate(lens):
            s = slice(at, at + n)
            _close(Y[s], X[s] @ W[e].T, np.abs(X[s]) @ np.abs(W[e].T), K, "bf16")
            _close(DX[s], D[s] @ W[e], np.abs(D[s]) @ np.abs(W[e]), N, "bf16")
            g = dw[e] if layout == LLAMA else dw[e].T
            _close(g, D[s].T @ X[s], np.abs(D[s]).T @ np.abs(X[s]), max(n, 1), "f32")
            at += n


def test_wide_strides_many_tiles(moe):
    # as many tiles as the larger tile sizes take
    print("grouped wide strides, many tiles", flush=True)
    rng = np.random.default_rng(17)
    E, K, N, ld = 64, 200, 200, 2**20 + 8
    M = 3 * E
    off = _offsets([3] * E)
    buf = torch.empty(M * ld, dtype=torch.float32, device="cuda")
    xw = buf.as_strided((M, K), (ld, 1))
    x, dy = _rows(rng, M, K, "f32", 0), _rows(rng, M, N, "f32", 0)
    xw.copy_(x)
    dw, X, D = _f64(moe.grouped_matmul_grad_w(xw, dy, off)), _f64(x), _f64(dy)
    for e in range(E):
        s = slice(3 * e, 3 * e + 3)
        _close(dw[e], D[s].T @ X[s], np.abs(D[s]).T @ np.abs(X[s]), 3, "f32")


def test_weight_matrices_past_2_31_elements(moe):
    print("grouped matrices past 2^31 elements", flush=True)
    rng = np.random.default_rng(13)
    E, N, K = 3, 40, 64
    stride = 2**30 + 64  # elements between the matrices: the last one starts past 2^31
    buf = torch.empty(2 * stride + N * K, dtype=torch.bfloat16, device="cuda")
    w = buf.as_strided((E, N, K), (stride, K, 1))
    w.copy_(_mats(rng, E, N, K, "bf16", 0))
    lens = [20, 70, 33]
    x, dy, off = _rows(rng, 123, K, "bf16", 0), _rows(rng, 123, N, "bf16", 0), _offsets(lens)
    W, dense = _f64(w), w.contiguous()
    assert torch.equal(moe.grouped_matmul(x, w, off), moe.grouped_matmul(x, dense, off))
    assert torch.equal(moe.grouped_matmul_grad_x(dy, w, off), moe.grouped_matmul_grad_x(dy, dense, off))
    dw = moe.grouped_matmul_grad_w(x, dy, off)
    X, D, at = _f64(x), _f64(dy), 0
    for e, n in enumerate(lens):
        _close(_f64(dw[e]), D[at:at + n].T @ X[at:at + n], np.abs(D[at:at + n]).T @ np.abs(X[at:at + n]), n, "bf16")
        at += n
    moe.grouped_matmul_grad_w(x, dy, off, out=w)
    assert torch.equal(w, dw)


@pytest.mark.parametrize("E", [500, 513, 1300])
def test_many_groups(moe, E):
    # the weight gradient's work list, longest group first, up to 512 groups and
    # past them; the row products' one, 64 groups at a time
    print(f"grouped many groups E={E}", flush=True)
    rng = np.random.default_rng(E)
    lens = [int(n) for n in rng.integers(0, 9, E)]
    lens[7], lens[E - 1] = 150, 0
    K, N, M = 40, 24, sum(lens)
    x, dy, w, off = _rows(rng, M, K, "bf16", 0), _rows(rng, M, N, "bf16", 0), _mats(rng, E, N, K, "bf16", 0), _offsets(lens)
    y, dx, dw = moe.grouped_matmul(x, w, off), moe.grouped_matmul_grad_x(dy, w, off), moe.grouped_matmul_grad_w(x, dy, off)
    X, D, W, Y, DX, DW, at = _f64(x), _f64(dy), _f64(w), _f64(y), _f64(dx), _f64(dw), 0
    for e, n in enumerate(lens):
        s = slice(at, at + n)
        _close(Y[s], X[s] @ W[e].T, np.abs(X[s]) @ np.abs(W[e].T), K, "bf16")
        _close(DX[s], D[s] @ W[e], np.abs(D[s]) @ np.abs(W[e]), N, "bf16")
        _close(DW[e], D[s].T @ X[s], np.abs(D[s]).T @ np.abs(X[s]), max(n, 1), "bf16")
        at += n


def test_two_streams_at_once(moe):
    # calls that run side by side on two streams, split ones (each with its own
    # workspace) among them: the bits of the calls alone
    rng = np.random.default_rng(14)
    jobs = []
    for lens, K, N in (([71], 5440, 64), ([3, 0, 2], 16401, 125), ([3000], 96, 40), ([33, 130, 5, 0, 300], 200, 136)):
        x, dy = _rows(rng, sum(lens), K, "bf16", 0), _rows(rng, sum(lens), N, "bf16", 0)
        w, off = _mats(rng, len(lens), N, K, "bf16", 0), _offsets(lens)
        jobs.append((x, dy, w, off))

    def run(i):
        x, dy, w, off = jobs[i]
        return (moe.grouped_matmul(x, w, off), moe.grouped_matmul_grad_x(dy, w, off), moe.grouped_matmul_grad_w(x, dy, off))

    want = [run(i) for i in range(len(jobs))]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(((turn + k) % len(jobs), run((turn + k) % len(jobs))))
    torch.cuda.synchronize()
    for i, res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want[i])), i


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_weight_gradient_of_two_rounds_of_large_tiles(moe, layout):
    # four groups of 8 x 16 tiles of 256 x 256: as many as take that size
    rng = np.random.default_rng(19)
    lens, K, N = [70, 0, 133, 9], 4096, 2040
    x, dy = _rows(rng, 212, K, "bf16", 0), _rows(rng, 212, N, "bf16", 0)
    dw = moe.grouped_matmul_grad_w(x, dy, _offsets(lens), layout=layout, out_dtype=torch.float32)
    a, b = (_f64(dy), _f64(x)) if layout == LLAMA else (_f64(x), _f64(dy))
    for e, s in enumerate((slice(0, 70), slice(70, 70), slice(70, 203), slice(203, 212))):
        _close(_f64(dw[e]), a[s].T @ b[s], np.abs(a[s]).T @ np.abs(b[s]), max(lens[e], 1), "f32")


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_sums_of_more_than_half_a_tile_per_cu(moe, dtype, layout):
    # k split over workgroups where 64 x 64 tiles alone fill more than half of the GPU
    K = {"f32": 3101, "bf16": 5440}[dtype]
    for lens, N in (([200], 2500), ([150, 0, 77, 1], 1800), ([130], 8200)):
        print(f"grouped split of many tiles {dtype} layout={layout} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, 6])
        M, E, start = sum(lens), len(lens), 1
        x = _rows(rng, M + start, K, dtype, 0, 2)
        w = _mats(rng, E, *((N, K) if layout == LLAMA else (K, N)), dtype, 0)
        W, X = (_f64(w) if layout == LLAMA else _f64(w).transpose(0, 2, 1)), _f64(x)
        out = torch.full((M + start + 2, N + 2), SENTINEL, dtype=DT[dtype], device="cuda")
        got, at = _f64(moe.grouped_matmul(x, w, _offsets(lens, start), layout=layout, out=out[:, :N])), start
        for e, n in enumerate(lens):
            a = X[at:at + n]
            _close(got[at:at + n], a @ W[e].T, np.abs(a) @ np.abs(W[e].T), K, dtype)
            at += n
        assert (got[:start] == SENTINEL).all() and (got[at:] == SENTINEL).all() and (_f64(out)[:, N:] == SENTINEL).all()


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_long_weight_gradients_of_more_than_half_a_tile_per_cu(moe, layout):
    for lens, K, N in (([4100], 1030, 1000), ([6000, 0, 7001], 330, 700)):
        print(f"grad_w split of many tiles layout={layout} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, 7])
        M = sum(lens)
        x, dy, off = _rows(rng, M, K, "f32", 0), _rows(rng, M, N, "f32", 0), _offsets(lens)
        a, b = (_f64(dy), _f64(x)) if layout == LLAMA else (_f64(x), _f64(dy))
        out = torch.ones(len(lens), a.shape[1], b.shape[1], device="cuda")
        moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out=out, accumulate=True)
        got, at = _f64(out), 0
        for e, n in enumerate(lens):
            s = slice(at, at + n)
            _close(got[e], 1 + a[s].T @ b[s], 1 + np.abs(a[s]).T @ np.abs(b[s]), max(n, 1) + 1, "f32")
            at += n


def test_two_graphs_of_split_sums(moe):
    # calls with workspaces in two captured graphs, replayed in turn and side by side
    # with eager calls of the same between them
    rng = np.random.default_rng(20)
    jobs = []
    for dtype, lens, K, N in (("f32", [150, 0, 77], 3101, 1800), ("bf16", [200], 5440, 2500), ("f32", [3000, 1], 96, 40)):
        x, dy = _rows(rng, sum(lens), K, dtype, 0), _rows(rng, sum(lens), N, dtype, 0)
        jobs.append((x, dy, _mats(rng, len(lens), N, K, dtype, 0), _offsets(lens)))

    def run(xs):
        return [f for x, (_, dy, w, off) in zip(xs, jobs)
                for f in (moe.grouped_matmul(x, w, off), moe.grouped_matmul_grad_w(x, dy, off))]

    first = [j[0] for j in jobs]
    sets = [first, [x * 2 for x in first], [x * -0.5 for x in first]]
    want = [run(s) for s in sets]
    bufs = [[x.clone() for x in first] for _ in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(b))
        graphs.append(g)
    side = torch.cuda.Stream()
    for i, k in ((0, 1), (1, 2), (2, 0), (1, 1)):
        for b, n in zip(bufs, (i, k)):
            for x, v in zip(b, sets[n]):
                x.copy_(v)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        eager = run(sets[k])
        torch.cuda.synchronize()
        for got, n in ((outs[0], i), (outs[1], k), (eager, k)):
            assert all(torch.equal(a, b) for a, b in zip(got, want[n])), (i, k)
