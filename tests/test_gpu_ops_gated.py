"""gated_matmul and its gradients (ops.py) against float64 of the same inputs.

Tolerance per element.  A sum of K products in fp32 is off by at most K * 2^-23 of
the sum of their magnitudes (sums below: d).  The gate: with z the sigmoid's
argument, e^-z is off by 2^-22 (|z| + 8) of itself (the argument's roundings, times
|z|, and the exponential's, the sum's and the reciprocal's own), which bounds the
relative error of act(a) and, times s + |a| s g, the absolute one of act'(a) = s +
a s (1 - s) g (silu: g = 1; gelu: g = r (1 + 3 c a^2)).  A sum's error passes through
act with |act'| <= 1.13 (gelu's largest slope; silu's is 1.1).  Then one rounding to
the result's type, half a step: 2^-8 of a bf16 value, 2^-24 of an fp32 one."""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FLUX, LLAMA = 0, 1
SENTINEL = 776.0  # exact in bf16 and fp32
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = {"bf16": 2.0**-8, "f32": 2.0**-24}
ACTS = ["silu", "gelu", "relu", "identity"]


def _rows(rng, rows, cols, dtype, pad=0, tail=0, scale=1.0):
    """rows + tail rows of a wider tensor; the padding columns and the rows past the
    groups hold NaN."""
    t = torch.full((rows + tail, cols + pad), float("nan"), dtype=DT[dtype])
    t[:rows, :cols] = torch.from_numpy(rng.standard_normal((rows, cols)) * scale).to(DT[dtype])
    return t.cuda()[:, :cols]


def _mats(rng, E, out_dim, in_dim, dtype, layout, pad=0):
    a, b = (out_dim, in_dim) if layout == LLAMA else (in_dim, out_dim)
    t = torch.full((E, a, b + pad), float("nan"), dtype=DT[dtype])
    t[:, :, :b] = torch.from_numpy(rng.standard_normal((E, a, b)) * in_dim**-0.5).to(DT[dtype])
    return t.cuda()[:, :, :b]


def _f64(t):
    return t.detach().cpu().double().numpy()


def _out_in(w, layout):
    return _f64(w) if layout == LLAMA else _f64(w).transpose(0, 2, 1)


def _offsets(lens, start=0):
    return torch.tensor(np.concatenate([[start], start + np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _gate(act, a):
    """act(a), act'(a), the relative error of the first and the absolute one of the second."""
    if act == "relu":
        return np.maximum(a, 0), (a > 0) * 1.0, 0.0, 0.0
    if act == "identity":
        return a, np.ones_like(a), 0.0, 0.0
    r, c = 2 * np.sqrt(2 / np.pi), 0.044715
    z, g = (a, np.ones_like(a)) if act == "silu" else (r * (a + c * a**3), r * (1 + 3 * c * a * a))
    with np.errstate(over="ignore"):
        s, t = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    e = 2.0**-22 * (np.abs(z) + 8)
    return a * s, s + a * s * t * g, e, e * (s + np.abs(a) * s * g)


def _near(got, ref, tol, dtype, what):
    tol = tol + np.abs(ref) * STEP[dtype] + 1e-35
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - ref)[bad].max()), float(tol[bad].max()))


def _groups(lens, at=0):
    for e, n in enumerate(lens):
        yield e, slice(at, at + n)
        at += n


def _check_forward(lens, act, got, x, w1, w3, layout, K, dtype, odt, start=0):
    """got: h, or (h, a, b), as numpy."""
    X, W1, W3 = _f64(x), _out_in(w1, layout), _out_in(w3, layout)
    for e, s in _groups(lens, start):
        a, b = X[s] @ W1[e].T, X[s] @ W3[e].T
        mag = np.abs(X[s])
        da, db = (K * 2.0**-23 * (mag @ np.abs(w[e].T)) for w in (W1, W3))
        f, _, err, _ = _gate(act, a)
        h = f * b
        _near(got[0][s], h, 1.13 * da * (np.abs(b) + db) + np.abs(f) * db + np.abs(h) * (err + 2.0**-23), odt, "h")
        if len(got) > 1:
            _near(got[1][s], a, da, dtype, "a")
            _near(got[2][s], b, db, dtype, "b")


def _check_grad(lens, act, got, dy, a, b, w2, layout, K, dtype, start=0):
    D, A, B = _f64(dy), _f64(a), _f64(b)
    W2 = None if w2 is None else _out_in(w2, layout)
    for e, s in _groups(lens, start):
        dh = D[s] if W2 is None else D[s] @ W2[e]
        d = 0 if W2 is None else K * 2.0**-23 * (np.abs(D[s]) @ np.abs(W2[e]))
        f, g, ef, eg = _gate(act, A[s])
        da, db, h = dh * B[s] * g, dh * f, f * B[s]
        _near(got[0][s], da, (d * np.abs(g) + (np.abs(dh) + d) * eg) * np.abs(B[s]) + np.abs(da) * 2.0**-22, dtype, "da")
        _near(got[1][s], db, d * np.abs(f) * (1 + ef) + np.abs(db) * (ef + 2.0**-23), dtype, "db")
        _near(got[2][s], h, np.abs(h) * (ef + 2.0**-23), dtype, "h")


def _check_grad_x(lens, got, da, db, w1, w3, layout, H, odt, start=0):
    A, B, W1, W3 = _f64(da), _f64(db), _out_in(w1, layout), _out_in(w3, layout)
    for e, s in _groups(lens, start):
        mag = np.abs(A[s]) @ np.abs(W1[e]) + np.abs(B[s]) @ np.abs(W3[e])
        _near(got[s], A[s] @ W1[e] + B[s] @ W3[e], 2 * H * 2.0**-23 * mag, odt, "dx")


# group lengths, K, H: no rows, one row, odd sizes below, at and past the tiles' edges
SHAPES = [
    ([1], 1, 1),
    ([0, 3, 0], 7, 5),
    ([17, 0, 1, 64], 64, 96),
    ([33, 130, 5, 0, 300], 200, 136),
    ([16, 16, 31, 2], 129, 257),
    ([70, 90, 65], 333, 72),
    ([0, 0], 40, 24),
    ([5] * 70, 96, 48),              # more groups than a wave has lanes
    ([700, 0, 900, 500], 72, 1024),  # 128 x 128 tiles
]


def _empty(rows, cols, pad, dtype):
    whole = torch.full((rows, cols + pad), SENTINEL, dtype=DT[dtype], device="cuda")
    return whole, whole[:, :cols]


def _untouched(wholes, cols, M):
    for t in wholes:
        t = _f64(t)
        assert (t[M:] == SENTINEL).all() and (t[:, cols:] == SENTINEL).all()


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_forward(moe, dtype, odt, layout, pad):
    for i, (lens, K, H) in enumerate(SHAPES):
        act = ACTS[(i + pad) % 4]
        print(f"gated {dtype}->{odt} {act} layout={layout} pad={pad} lens={lens[:6]} K={K} H={H}", flush=True)
        rng = np.random.default_rng([K, H, layout, pad])
        M, E, tail = sum(lens), len(lens), 5
        x = _rows(rng, M, K, dtype, pad, tail)
        w1, w3 = (_mats(rng, E, H, K, dtype, layout, p) for p in (pad, 0))
        wholes, views = zip(*(_empty(M + tail, H, pad, t) for t in (odt, dtype, dtype)))
        kw = dict(activation=getattr(moe, act), layout=layout)
        res = moe.gated_matmul(x, w1, w3, _offsets(lens), save=True, out=views, **kw)
        assert all(r is v for r, v in zip(res, views))
        _check_forward(lens, act, [_f64(t) for t in res], x, w1, w3, layout, K, dtype, odt)
        _untouched(wholes, H, M)
        # without a and b: the same h
        whole, view = _empty(M + tail, H, 0, odt)
        assert moe.gated_matmul(x, w1, w3, _offsets(lens), out=view, **kw) is view
        assert torch.equal(view, views[0])


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients(moe, dtype, layout, pad):
    for i, (lens, K, H) in enumerate(SHAPES):
        act = ACTS[(i + pad) % 4]
        print(f"gated gradients {dtype} {act} layout={layout} pad={pad} lens={lens[:6]} K={K} H={H}", flush=True)
        rng = np.random.default_rng([K, H, layout, pad, 1])
        M, E, tail, off = sum(lens), len(lens), 5, _offsets(lens)
        a, b = _rows(rng, M, H, dtype, pad, tail, 2.0), _rows(rng, M, H, dtype, 0, tail)
        w2 = _mats(rng, E, K, H, dtype, layout, pad)
        for w, dy in ((w2, _rows(rng, M, K, dtype, pad, tail)), (None, _rows(rng, M, H, dtype, 0, tail))):
            wholes, views = zip(*(_empty(M + tail, H, p, dtype) for p in (pad, 0, 1)))
            res = moe.gated_matmul_grad(dy, a, b, w, off, activation=getattr(moe, act), layout=layout, out=views)
            assert all(r is v for r, v in zip(res, views))
            _check_grad(lens, act, [_f64(t) for t in res], dy, a, b, w, layout, K, dtype)
            _untouched(wholes, H, M)
        da, db = _rows(rng, M, H, dtype, pad, tail), _rows(rng, M, H, dtype, 0, tail)
        w1, w3 = (_mats(rng, E, H, K, dtype, layout, p) for p in (pad, 0))
        whole, view = _empty(M + tail, K, pad, dtype)
        assert moe.gated_matmul_grad_x(da, db, w1, w3, off, layout=layout, out=view) is view
        _check_grad_x(lens, _f64(view), da, db, w1, w3, layout, H, dtype)
        _untouched([whole], K, M)


@pytest.mark.parametrize("dtype,K,most", [("f32", 200, 32), ("f32", 1024, 32), ("f32", 1032, 64), ("bf16", 200, 64)])
def test_few_rows_in_uneven_groups(moe, dtype, K, most):
    """Streamed, by the average of rows: the groups of more are taken in parts."""
    lens, H, tail = [70, 1, 0, 33, 0, 0, 16] + [0] * 9, 72, 3
    rng = np.random.default_rng(K)
    x = _rows(rng, sum(lens), K, dtype, 8, tail)
    w1, w3 = _mats(rng, len(lens), H, K, dtype, LLAMA, 8), _mats(rng, len(lens), H, K, dtype, LLAMA)
    res, off = [], _offsets(lens)
    names = kernels_of(lambda: res.append(moe.gated_matmul(x, w1, w3, off, save=True)))
    assert names["op_gated_stream_kernel"][1] == str(most)
    _check_forward(lens, "silu", [_f64(t) for t in res[0]], x, w1, w3, LLAMA, K, dtype, dtype)
    assert not any(t[sum(lens):].any() for t in res[0])


def _tile(names, mode):
    """Rows of the tiles and alignment of the loads of the call's gated kernel."""
    a = names["op_gated_kernel"]
    assert int(a[0]) == mode, names
    return int(a[3]), int(a[10])


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_large_tiles(moe, layout):
    # 256 x 256 tiles, ragged last tiles, k with a part stage; strides that differ
    rng = np.random.default_rng(5)
    lens, K, H = [2100, 1, 3000, 3400], 136, 2024
    M, off = sum(lens), _offsets(lens)
    x, w1, w3 = _rows(rng, M, K, "bf16"), _mats(rng, 4, H, K, "bf16", layout), _mats(rng, 4, H, K, "bf16", layout, 8)
    print(f"gated 256-row tiles layout={layout}", flush=True)
    res = []
    names = kernels_of(lambda: res.append(moe.gated_matmul(x, w1, w3, off, layout=layout, save=True)))
    assert _tile(names, 1) == (256, 16)
    _check_forward(lens, "silu", [_f64(t) for t in res[-1]], x, w1, w3, layout, K, "bf16", "bf16")
    for act in ACTS[1:]:
        h = moe.gated_matmul(x, w1, w3, off, layout=layout, activation=getattr(moe, act), out_dtype=torch.float32)
        _check_forward(lens, act, [_f64(h)], x, w1, w3, layout, K, "bf16", "f32")
    dy, w2 = _rows(rng, M, K, "bf16", 8), _mats(rng, 4, K, 2 * H, "bf16", layout)
    a, b = _rows(rng, M, 2 * H, "bf16"), _rows(rng, M, 2 * H, "bf16", 8)
    names = kernels_of(lambda: res.append(moe.gated_matmul_grad(dy, a, b, w2, off, layout=layout)))
    assert _tile(names, 2) == (256, 16)
    _check_grad(lens, "silu", [_f64(t) for t in res[-1]], dy, a, b, w2, layout, K, "bf16")
    for act in ACTS[1:]:
        grads = moe.gated_matmul_grad(dy, a, b, w2, off, layout=layout, activation=getattr(moe, act))
        _check_grad(lens, act, [_f64(t) for t in grads], dy, a, b, w2, layout, K, "bf16")
    # the two pairs' strides alike: 256 x 256 tiles; apart: 128 x 128
    for p, q, rows in ((0, 0, 256), (8, 0, 128), (0, 8, 128)):
        Kx, Hx = 4040, 104
        da, db = _rows(rng, M, Hx, "bf16"), _rows(rng, M, Hx, "bf16", p)
        v1, v3 = _mats(rng, 4, Hx, Kx, "bf16", layout), _mats(rng, 4, Hx, Kx, "bf16", layout, q)
        names = kernels_of(lambda: res.append(moe.gated_matmul_grad_x(da, db, v1, v3, off, layout=layout)))
        assert _tile(names, 3) == (rows, 16)
        _check_grad_x(lens, _f64(res[-1]), da, db, v1, v3, layout, Hx, "bf16")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_form_of_every_activation(moe, dtype, act):
    # 64 x 64 and 128 x 128 tiles and the streamed form, each load form, both orders
    for lens, K, H, layout in (([40, 0, 33], 64, 72, LLAMA), ([40, 0, 33], 66, 74, FLUX), ([40, 0, 33], 65, 73, LLAMA),
                               ([3, 0, 1], 64, 72, LLAMA), ([700, 0, 900, 500], 72, 1024, LLAMA),
                               ([700, 0, 900, 500], 74, 1026, FLUX), ([700, 0, 900, 500], 73, 1025, FLUX)):
        rng = np.random.default_rng([K, H, layout, 4])
        M, off, fn = sum(lens), _offsets(lens), getattr(moe, act)
        x, w1, w3 = _rows(rng, M, K, dtype), *(_mats(rng, len(lens), H, K, dtype, layout) for _ in range(2))
        print(f"gated forms {dtype} {act} lens={lens} K={K} H={H} layout={layout}", flush=True)
        res = moe.gated_matmul(x, w1, w3, off, activation=fn, layout=layout, save=True)
        _check_forward(lens, act, [_f64(t) for t in res], x, w1, w3, layout, K, dtype, dtype)
        w2, dy = _mats(rng, len(lens), K, H, dtype, layout), _rows(rng, M, K, dtype)
        grads = moe.gated_matmul_grad(dy, res[1], res[2], w2, off, activation=fn, layout=layout)
        _check_grad(lens, act, [_f64(t) for t in grads], dy, res[1], res[2], w2, layout, K, dtype)


def test_many_groups(moe):
    # more groups than rows, and more than a wave's scan; rows behind the last one
    rng = np.random.default_rng(18)
    E, K, H = 700, 32, 24
    lens = [int(v) for v in rng.integers(0, 3, E)]
    M, off = sum(lens), _offsets(lens)
    x, w1, w3 = _rows(rng, M, K, "bf16", 0, 9), *(_mats(rng, E, H, K, "bf16", LLAMA) for _ in range(2))
    h, a, b = moe.gated_matmul(x, w1, w3, off, save=True)
    _check_forward(lens, "silu", [_f64(t) for t in (h, a, b)], x, w1, w3, LLAMA, K, "bf16", "bf16")
    dx = moe.gated_matmul_grad_x(a, b, w1, w3, off)
    _check_grad_x(lens, _f64(dx), a, b, w1, w3, LLAMA, H, "bf16")
    assert (h[M:] == 0).all() and (dx[M:] == 0).all()


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("lens", [[1500, 700, 1896], [1025, 1025, 2046], [2048, 0, 2048]])
def test_split_last_round(moe, lens, layout):
    # two rounds of 256 x 256 tiles and a part of one, whose tiles are split; or none
    rng = np.random.default_rng(16)
    K, H = 8184, 4100 if layout == FLUX else 4104
    H = H // 8 * 8
    M, off = sum(lens), _offsets(lens)
    g = torch.Generator(device="cuda").manual_seed(7)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    da, db = new(M + 3, H), new(M + 3, H)
    shape = (3, H, K) if layout == LLAMA else (3, K, H)
    w1, w3 = new(*shape), new(*shape)
    for odt in ("bf16", "f32"):
        whole, view = _empty(M + 3, K, 0, odt)
        names = kernels_of(lambda: moe.gated_matmul_grad_x(da, db, w1, w3, off, layout=layout, out=view))
        assert _tile(names, 3) == (256, 16) and "op_tail_fold_kernel" in names
        for e, s in _groups(lens):  # float64 on the GPU: 5e11 products
            m1, m3 = ((w[e] if layout == LLAMA else w[e].t()).double() for w in (w1, w3))
            a, b = da[s].double(), db[s].double()
            ref, mag = a @ m1 + b @ m3, a.abs() @ m1.abs() + b.abs() @ m3.abs()
            assert ((view[s].double() - ref).abs() <= 2 * H * 2.0**-23 * mag + ref.abs() * STEP[odt]).all()
        assert (view[M:] == SENTINEL).all()


# few rows and columns of a long sum: k split over workgroups, streamed and tiled
LONG = [([1], 8192, 16), ([3, 0, 2], 4001, 125), ([3, 0, 2], 16401, 45), ([71], 5440, 64), ([200, 0, 150], 3456, 131),
        ([40, 3], 2999, 64)]


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("dtype,odt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_long_sums(moe, dtype, odt, layout):
    folds = 0
    for lens, K, N in LONG:
        print(f"gated long sum {dtype}->{odt} layout={layout} lens={lens} K={K} N={N}", flush=True)
        rng = np.random.default_rng([K, N, layout, 2])
        M, E, start, tail = sum(lens), len(lens), 2, 4
        off, rows = _offsets(lens, start), sum(lens) + start
        act = moe.gelu
        x, w1, w3 = _rows(rng, rows, K, dtype, 0, tail), _mats(rng, E, N, K, dtype, layout), _mats(rng, E, N, K, dtype, layout)
        wholes, views = zip(*(_empty(rows + tail, N, 3, t) for t in (odt, dtype, dtype)))
        names = kernels_of(lambda: moe.gated_matmul(x, w1, w3, off, activation=act, layout=layout, save=True, out=views))
        folds += any("fold" in n for n in names)
        _check_forward(lens, "gelu", [_f64(t) for t in views], x, w1, w3, layout, K, dtype, odt, start)
        if odt == dtype:
            w2, dy = _mats(rng, E, K, N, dtype, layout), _rows(rng, rows, K, dtype, 0, tail)
            a, b = _rows(rng, rows, N, dtype, 0, tail), _rows(rng, rows, N, dtype, 0, tail)
            grads, gviews = zip(*(_empty(rows + tail, N, 3, dtype) for _ in range(3)))
            names = kernels_of(lambda: moe.gated_matmul_grad(dy, a, b, w2, off, activation=act, layout=layout, out=gviews))
            folds += any("fold" in n for n in names)
            _check_grad(lens, "gelu", [_f64(t) for t in gviews], dy, a, b, w2, layout, K, dtype, start)
            wholes += grads
        # a long hidden size for the row gradient, both pairs' ends inside ranges
        v1, v3 = _mats(rng, E, K, N, dtype, layout), _mats(rng, E, K, N, dtype, layout, 16)
        da, db = _rows(rng, rows, K, dtype, 0, tail), _rows(rng, rows, K, dtype, 8, tail)
        whole, view = _empty(rows + tail, N, 3, odt)
        names = kernels_of(lambda: moe.gated_matmul_grad_x(da, db, v1, v3, off, layout=layout, out=view))
        folds += any("fold" in n for n in names)
        _check_grad_x(lens, _f64(view), da, db, v1, v3, layout, K, odt, start)
        for t in wholes + (whole,):
            t = _f64(t)
            assert (t[:start] == SENTINEL).all() and (t[rows:] == SENTINEL).all() and (t[:, N:] == SENTINEL).all()
    assert folds >= 9


def test_forms(moe):
    # few rows: streamed where the weights are rows; loads by alignment
    for lens, K, H, dtype, layout, form in (([1, 0, 3], 64, 96, "bf16", LLAMA, "op_gated_stream_kernel"),
                                           ([1, 0, 3], 64, 96, "bf16", FLUX, (64, 16)),
                                           ([16, 16], 64, 96, "f32", LLAMA, "op_gated_stream_kernel"),
                                           ([40, 16], 202, 134, "bf16", LLAMA, (64, 4)),
                                           ([40, 16], 201, 135, "bf16", LLAMA, (64, 0)),
                                           ([40, 16], 201, 135, "f32", FLUX, (64, 4))):
        rng = np.random.default_rng(1)
        x, off = _rows(rng, sum(lens), K, dtype), _offsets(lens)
        w1, w3 = (_mats(rng, len(lens), H, K, dtype, layout) for _ in range(2))
        names = kernels_of(lambda: moe.gated_matmul(x, w1, w3, off, layout=layout))
        if isinstance(form, str):
            assert form in names and "op_gated_kernel" not in names
        else:
            assert _tile(names, 1) == form


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_wide_strides(moe, dtype):
    # rows 4 MB apart and more: through registers, offsets past 32 bits
    rng = np.random.default_rng(7)
    ld = (1 << 20) + 4 if dtype == "f32" else (1 << 21) + 8
    K, H, rows = 24, 40, 600
    big = torch.zeros(rows, ld, dtype=DT[dtype], device="cuda")
    put = lambda at, t: big[:t.shape[0], at:at + t.shape[1]].copy_(t)
    x = put(0, _rows(rng, rows, K, dtype))
    off, w1, w3 = _offsets([500, 0, 100]), *(_mats(rng, 3, H, K, dtype, LLAMA) for _ in range(2))
    w2 = _mats(rng, 3, K, H, dtype, LLAMA)
    out = tuple(big[:, 100 * i:100 * i + H] for i in (1, 2, 3))
    h, a, b = moe.gated_matmul(x, w1, w3, off, save=True, out=out)
    _check_forward([500, 0, 100], "silu", [_f64(t) for t in (h, a, b)], x, w1, w3, LLAMA, K, dtype, dtype)
    dy = put(500, _rows(rng, rows, K, dtype))
    grads = moe.gated_matmul_grad(dy, a, b, w2, off, out=tuple(big[:, 600 + 100 * i:600 + 100 * i + H] for i in range(3)))
    _check_grad([500, 0, 100], "silu", [_f64(t) for t in grads], dy, a, b, w2, LLAMA, K, dtype)
    dx = moe.gated_matmul_grad_x(grads[0], grads[1], w1, w3, off, out=big[:, 1000:1000 + K])
    _check_grad_x([500, 0, 100], _f64(dx), grads[0], grads[1], w1, w3, LLAMA, H, dtype)


def test_one_expert_and_defaults(moe):
    rng = np.random.default_rng(8)
    x, w1, w3 = _rows(rng, 50, 24, "bf16"), *(_mats(rng, 1, 40, 24, "bf16", LLAMA) for _ in range(2))
    h = moe.gated_matmul(x, w1[0], w3[0], out_dtype=torch.float32)
    assert h.dtype == torch.float32 and h.shape == (50, 40)
    _check_forward([50], "silu", [_f64(h)], x, w1, w3, LLAMA, 24, "bf16", "f32")
    # both weights in one buffer, as (E, 2 hidden, in)
    both = torch.cat([w1, w3], dim=1)
    assert torch.equal(moe.gated_matmul(x, both[:, :40], both[:, 40:], out_dtype=torch.float32), h)
    # rows outside every group, when the call makes the results: zeros
    off = torch.tensor([10, 30], dtype=torch.int32, device="cuda")
    h, a, b = moe.gated_matmul(x, w1, w3, off, save=True)
    grads = moe.gated_matmul_grad(x, a, b, w1.transpose(1, 2).contiguous(), off)
    own = moe.gated_matmul_grad(h, a, b, None, off)
    dx = moe.gated_matmul_grad_x(grads[0], grads[1], w1, w3, off)
    for t in (h, a, b, dx, *grads, *own):
        assert (t[:10] == 0).all() and (t[30:] == 0).all() and (t[10:30] != 0).any()
    # no rows at all
    none = moe.gated_matmul(x[:0], w1, w3, _offsets([0]), save=True)
    assert [t.shape for t in none] == [(0, 40)] * 3
    assert [t.shape for t in moe.gated_matmul_grad(x[:0], none[1], none[2], w1.transpose(1, 2).contiguous())] == [(0, 40)] * 3
    assert moe.gated_matmul_grad(none[0], none[1], none[2])[0].shape == (0, 40)
    assert moe.gated_matmul_grad_x(none[1], none[2], w1, w3, _offsets([0])).shape == (0, 24)


def test_infinities_stay_in_their_rows(moe):
    rng = np.random.default_rng(9)
    off = _offsets([100, 100])
    x, w1, w3 = _rows(rng, 200, 72, "bf16"), *(_mats(rng, 2, 72, 72, "bf16", LLAMA) for _ in range(2))
    x[5, 3], x[150, 71] = float("inf"), float("nan")
    fin = lambda t: torch.isfinite(t).all(dim=1).cpu()
    h, a, b = moe.gated_matmul(x, w1, w3, off, save=True)
    for t in (h, a, b, *moe.gated_matmul_grad(x, b.nan_to_num(0, 0, 0), b.nan_to_num(0, 0, 0), w1, off)[:2],
              moe.gated_matmul_grad_x(x, x, w1, w3, off)):
        f = fin(t)
        assert not f[5] and not f[150] and f.sum() == 198


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_gate_far_out(moe, act, dtype):
    # the gate where its exponential overflows, underflows or its square would: act
    # is 0 (or a), its slope 0 (or 1), never NaN; NaN stays NaN
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20, -20, 87, -87, 90, -90, 200, -200, 1e4, -1e4, 1e13, -1e13, 1e20, -1e20,
                      1e38, -1e38, float("nan")], dtype=DT[dtype], device="cuda")[None].contiguous()
    one = torch.ones_like(v)
    da, db, h = moe.gated_matmul_grad(one, v, one, activation=getattr(moe, act))
    a = _f64(v)[0]
    f, g, ef, eg = _gate(act, np.clip(a, -1e5, 1e5))
    f = np.where(np.abs(a) > 1e5, np.where((a > 0) | (act == "identity"), a, 0.0), f)
    assert torch.isnan(db[0, -1]) and torch.isnan(h[0, -1])
    for t, ref, e in ((da, g, eg), (db, f, np.abs(f) * ef), (h, f, np.abs(f) * ef)):
        t = _f64(t)[0]
        assert np.isfinite(t[:-1]).all()
        # (below 2^-126 the hardware's exp may give 0)
        _near(t[:-1], ref[:-1], np.broadcast_to(np.asarray(e) + 2.0**-23 * np.abs(ref), ref.shape)[:-1] + 1e-33, dtype, act)


def test_offsets_out_of_range_stay_in_bounds(moe):
    rng = np.random.default_rng(10)
    x, w = _rows(rng, 40, 64, "bf16"), _mats(rng, 3, 64, 64, "bf16", LLAMA)
    off = torch.tensor([-5, 16, 1000, 2000], dtype=torch.int32, device="cuda")
    for o in (lambda o: moe.gated_matmul(x, w, w, o), lambda o: moe.gated_matmul_grad(x, x, x, w, o)[0],
              lambda o: moe.gated_matmul_grad(x, x, x, None, o)[0], lambda o: moe.gated_matmul_grad_x(x, x, w, w, o)):
        assert torch.equal(o(off), o(_offsets([16, 24, 0])))


class _Block(torch.autograd.Function):
    """y = W2 (act(W1 x) (W3 x)) per group, with the gradient calls in its backward."""

    @staticmethod
    def forward(ctx, moe, act, off, x, w1, w3, w2):
        h, a, b = moe.gated_matmul(x, w1, w3, off, activation=act, save=True)
        ctx.save_for_backward(x, w1, w3, w2, a, b)
        ctx.moe, ctx.act, ctx.off = moe, act, off
        return moe.grouped_matmul(h, w2, off)

    @staticmethod
    def backward(ctx, dy):
        moe, off = ctx.moe, ctx.off
        x, w1, w3, w2, a, b = ctx.saved_tensors
        dy = dy.contiguous()
        da, db, h = moe.gated_matmul_grad(dy, a, b, w2, off, activation=ctx.act)
        return (None, None, None, moe.gated_matmul_grad_x(da, db, w1, w3, off), moe.grouped_matmul_grad_w(x, da, off),
                moe.grouped_matmul_grad_w(x, db, off), moe.grouped_matmul_grad_w(h, dy, off))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_block_forward_and_backward(moe, act):
    # the chain as a training step uses it, against differences of the float64 formula
    rng = np.random.default_rng(13)
    lens, K, H, N = [9, 0, 20], 12, 20, 8
    M, off = sum(lens), _offsets(lens)
    ts = [_rows(rng, M, K, "f32"), _mats(rng, 3, H, K, "f32", LLAMA), _mats(rng, 3, H, K, "f32", LLAMA),
          _mats(rng, 3, N, H, "f32", LLAMA)]
    dy = _rows(rng, M, N, "f32")
    for t in ts:
        t.requires_grad_()
    y = _Block.apply(moe, getattr(moe, act), off, *ts)
    y.backward(dy)
    vals, D = [_f64(t) for t in ts], _f64(dy)

    def loss(x, w1, w3, w2):
        total = 0.0
        for e, s in _groups(lens):
            a, b = x[s] @ w1[e].T, x[s] @ w3[e].T
            total += (D[s] * ((_gate(act, a)[0] * b) @ w2[e].T)).sum()
        return total

    for i, t in enumerate(ts):
        grad = _f64(t.grad)
        for _ in range(40):
            at = tuple(rng.integers(0, n) for n in vals[i].shape)
            step = 1e-4
            up, down = [v.copy() for v in vals], [v.copy() for v in vals]
            up[i][at] += step
            down[i][at] -= step
            diff = (loss(*up) - loss(*down)) / (2 * step)
            # the difference: step^2 / 6 of a third derivative, at most about 30 here, and
            # 2^-52 of a loss of some tens over the step; the kernels: sums of up to 29
            # products of some units in fp32, three in a row
            assert abs(diff - grad[at]) <= 1e-4 * 1e-4 / 6 * 100 + 1e-9 + 3 * 29 * 2.0**-23 * 30, (i, at, diff, grad[at])
    assert (_f64(ts[1].grad)[1] == 0).all()  # an expert without rows


def test_streams_and_graph_replay(moe):
    # the bits of the calls alone: on another stream, two calls at once, and in every
    # replay of two captured graphs (split sums among the calls) with new inputs
    rng = np.random.default_rng(11)
    jobs = []
    for dtype, lens, K, H in (("bf16", [40, 0, 100, 77], 264, 136), ("bf16", [71], 5440, 64), ("f32", [3, 0, 2], 4001, 125)):
        E, M = len(lens), sum(lens)
        jobs.append((_rows(rng, M, K, dtype), _rows(rng, M, K, dtype), _mats(rng, E, H, K, dtype, LLAMA),
                     _mats(rng, E, H, K, dtype, LLAMA), _mats(rng, E, K, H, dtype, LLAMA), _offsets(lens)))

    def run(xs):
        out = []
        for x, (_, dy, w1, w3, w2, off) in zip(xs, jobs):
            h, a, b = moe.gated_matmul(x, w1, w3, off, save=True)
            grads = moe.gated_matmul_grad(dy, a, b, w2, off)
            out += [h, a, b, *grads, moe.gated_matmul_grad_x(grads[0], grads[1], w1, w3, off)]
        return out

    first = [j[0] for j in jobs]
    sets = [first, [x * 2 for x in first], [x * -0.5 for x in first]]
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
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    z = lambda n: torch.zeros(4, n, device="cuda")
    for outs, call in ((tuple(z(6) for _ in range(3)), lambda o: moe.gated_matmul(x, w, w, save=True, out=o)),
                       ((z(6),), lambda o: moe.gated_matmul(x, w, w, out=o[0])),
                       (tuple(z(8) for _ in range(3)), lambda o: moe.gated_matmul_grad(x, x, x, out=o)),
                       ((z(8),), lambda o: moe.gated_matmul_grad_x(z(6), z(6), w, w, out=o[0]))):
        before = [t._version for t in outs]
        call(outs)
        assert all(t._version > v for t, v in zip(outs, before))
