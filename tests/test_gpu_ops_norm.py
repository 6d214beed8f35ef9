"""block_norm and block_norm_grad (ops.py) against their formulas in float64,
and the gradients against differences.

Tolerances.  A sum over D channels in fp32 rounds by at most D 2^-24 of the sum
of magnitudes, in a tree of at most 16 + log2 steps here: rstd, from a sum of
squares of one sign, is good to 64 * 2^-24 =: E.  A forward value is a handful
of products of such factors: E of each term's magnitude, then half a step of
its type.  The reference takes the stored r (rounded to its type) as the kernel
gave it, so that a rounding tie decided the other way is not counted twice."""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8}
E = 64 * 2.0**-24
ALPHA, BETA, EPS = 0.75, -1.5, 1e-5


def _f64(t):
    return t.detach().cpu().double().numpy()


def _make(rng, shape, dt):
    return torch.from_numpy(rng.standard_normal(shape)).to(DT[dt]).cuda()


def _inputs(rng, T, D, xt, yt, wt, gates, pre, post, y=True):
    w = lambda on: _make(rng, D, wt) if on else None
    gate = None
    if gates:
        gate = _make(rng, (gates, D), xt)
    return dict(x=_make(rng, (T, D), xt), y=_make(rng, (T, D), yt) if y else None, pre_weight=w(pre),
                post_weight=w(post), gate=gate)


def _rstd(v, on):
    return (1.0 / np.sqrt((v * v).mean(axis=1, keepdims=True) + EPS)) if on else np.ones((v.shape[0], 1))


def _terms(a):
    """alpha x, beta gate z in float64."""
    x = ALPHA * _f64(a["x"])
    if a["y"] is None:
        return x, np.zeros_like(x)
    y = _f64(a["y"])
    z = y * _rstd(y, a["post_weight"] is not None)
    if a["post_weight"] is not None:
        z = z * _f64(a["post_weight"])
    if a["gate"] is not None:
        z = z * np.repeat(_f64(a["gate"]), x.shape[0] // a["gate"].shape[0], axis=0)
    return x, BETA * z


def _check_forward(moe, a, xt, ht):
    r, h, stats = moe.block_norm(a["x"], a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"],
                                 gate=a["gate"], alpha=ALPHA, beta=BETA, eps=EPS, h_dtype=DT[ht])
    x, z = _terms(a)
    tol = E * (np.abs(x) + np.abs(z)) + HALF[xt] * np.abs(x + z) + 1e-37
    assert (np.abs(_f64(r) - (x + z)) <= tol).all()
    if a["pre_weight"] is not None:
        R = _f64(r)
        ref = R * _rstd(R, True) * _f64(a["pre_weight"])
        assert h.dtype == DT[ht]
        assert (np.abs(_f64(h) - ref) <= (E + HALF[ht]) * np.abs(ref) + 1e-37).all()
        assert np.allclose(_f64(stats)[:, 1:], _rstd(R, True), rtol=E, atol=0)
    else:
        assert h is None
    if a["post_weight"] is not None:
        assert np.allclose(_f64(stats)[:, :1], _rstd(_f64(a["y"]), True), rtol=E, atol=0)
    return r, h, stats


def _formula(a, dr, dh, r):
    """(dx, dy, dgate, dpost, dpre), and the magnitudes that each one's terms have."""
    T, D = r.shape
    R, dr = _f64(r), _f64(dr) if dr is not None else np.zeros((T, D))
    G, mG, dpre, mpre = dr, np.abs(dr), None, None
    if a["pre_weight"] is not None:
        w, ir = _f64(a["pre_weight"]), _rstd(R, True)
        rh, t = R * ir, _f64(dh) * w
        dpre, mpre = (_f64(dh) * rh).sum(0), np.abs(_f64(dh) * rh).sum(0)
        G = dr + ir * (t - rh * (t * rh).mean(1, keepdims=True))
        mG = np.abs(dr) + ir * (np.abs(t) + np.abs(rh) * np.abs(t * rh).mean(1, keepdims=True))
    dx, mx = ALPHA * G, abs(ALPHA) * mG
    if a["y"] is None:
        return (dx, None, None, None, dpre), (mx, None, None, None, mpre)
    post = a["post_weight"] is not None
    y = _f64(a["y"])
    iy = _rstd(y, post)
    yh, wp = y * iy, _f64(a["post_weight"]) if post else np.ones(D)
    u, mu = BETA * G, abs(BETA) * mG
    dgate = mgate = None
    dz, mz = u, mu
    if a["gate"] is not None:
        n = a["gate"].shape[0]
        g = np.repeat(_f64(a["gate"]), T // n, axis=0)
        dgate, mgate = (u * yh * wp).reshape(n, T // n, D).sum(1), (mu * np.abs(yh * wp)).reshape(n, T // n, D).sum(1)
        dz, mz = u * g, mu * np.abs(g)
    dpost = mpost = None
    dy, my = dz, mz
    if post:
        dpost, mpost = (dz * yh).sum(0), (mz * np.abs(yh)).sum(0)
        b, mb = dz * wp, mz * np.abs(wp)
        dy = iy * (b - yh * (b * yh).mean(1, keepdims=True))
        my = iy * (mb + np.abs(yh) * (mb * np.abs(yh)).mean(1, keepdims=True))
    return (dx, dy, dgate, dpost, dpre), (mx, my, mgate, mpost, mpre)


def _check_grad(moe, a, r, stats, dr, dh, xt, yt):
    got = moe.block_norm_grad(dr, dh, r, a["y"], stats, pre_weight=a["pre_weight"], post_weight=a["post_weight"],
                              gate=a["gate"], alpha=ALPHA, beta=BETA)
    ref, mag = _formula(a, dr, dh, r)
    # dx, dy: a few factors of E each, sums over D; the column sums over T rows
    # add a rounding per row (at most T of them, in chunks)
    T = r.shape[0]
    for name, g, f, m, half in zip(("dx", "dy", "dgate", "dpost", "dpre"), got, ref, mag,
                                   (HALF[xt], HALF[yt], 2.0**-24, 2.0**-24, 2.0**-24)):
        if f is None:
            assert g is None, name
            continue
        tol = (4 * E + (T * 2.0**-24 if name[1:] not in ("x", "y") else 0.0)) * m + half * np.abs(f) + 1e-37
        bad = ~(np.abs(_f64(g).reshape(f.shape) - f) <= tol)
        assert not bad.any(), (name, int(bad.sum()))
    return got


SIZES = [(1, 1), (3, 7), (1, 512), (5, 520), (4, 1000), (66, 96), (2, 2048), (3, 2056), (4, 4096), (2, 5000), (3, 8192),
         (2, 9001), (6, 16384), (700, 64), (130, 1024)]


@pytest.mark.parametrize("xt,yt,ht,wt", [("f32", "f32", "f32", "f32"), ("bf16", "f32", "bf16", "f32"),
                                         ("bf16", "bf16", "bf16", "bf16"), ("f32", "bf16", "bf16", "f32"),
                                         ("bf16", "bf16", "f32", "f32")])
def test_sizes(moe, xt, yt, ht, wt):
    for T, D in SIZES:
        for gates in (0, 1, T):
            print(f"norm {xt}/{yt}/{ht}/{wt} T={T} D={D} gates={gates}", flush=True)
            rng = np.random.default_rng([T, D, gates])
            a = _inputs(rng, T, D, xt, yt, wt, gates, True, True)
            r, h, stats = _check_forward(moe, a, xt, ht)
            _check_grad(moe, a, r, stats, _make(rng, (T, D), xt), _make(rng, (T, D), ht), xt, yt)


def test_parts(moe):
    # every combination of the optional parts, gates shared by 1, 2, 7 and 35 rows
    T, D = 70, 72
    for pre, post, gates, y, hasdr in itertools.product((True, False), (True, False), (0, 1, 2, 10, 35, 70), (True, False),
                                                        (True, False)):
        if not y and (post or gates or not pre) or not (hasdr or pre) or not (pre or y):
            continue
        print(f"norm parts pre={pre} post={post} gates={gates} y={y} dr={hasdr}", flush=True)
        rng = np.random.default_rng(gates)
        a = _inputs(rng, T, D, "bf16", "f32", "f32", gates, pre, post, y)
        r, h, stats = _check_forward(moe, a, "bf16", "bf16")
        dr = _make(rng, (T, D), "bf16") if hasdr else None
        _check_grad(moe, a, r, stats, dr, _make(rng, (T, D), "bf16") if pre else None, "bf16", "f32")


@pytest.mark.parametrize("D", [1000, 2056, 6000, 16384])
@pytest.mark.parametrize("post", [False, True])
def test_many_rows_of_one_sum(moe, D, post):
    # only one of the two norms: the waves of a workgroup meet once per row, and
    # each workgroup takes several rows in turn
    T = 600
    print(f"norm one sum per row D={D} post={post}", flush=True)
    rng = np.random.default_rng([D, post])
    a = _inputs(rng, T, D, "bf16", "f32", "f32", 0, not post, post, y=post)
    r, h, stats = moe.block_norm(a["x"], a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"], alpha=ALPHA,
                                 beta=BETA, eps=EPS)
    dr = _make(rng, (T, D), "bf16") if post else None
    dh = None if post else _make(rng, (T, D), "bf16")
    _check_grad(moe, a, r, stats, dr, dh, "bf16", "f32")


@pytest.mark.parametrize("T,D,yt,gates", [(300, 1000, "f32", 300), (200, 4096, "bf16", 0), (60, 12000, "f32", 60), (900, 328, "f32", 1)])
def test_bf16_stream_with_an_fp32_norm(moe, T, D, yt, gates):
    # r is the float64 formula's value rounded by way of fp32, but for values whose
    # sum of squares decides the border: per thread at most 32 squares are added in
    # fp32, so rstd is off by at most 16 * 2^-24, which moves a bf16 border (2^-8
    # apart, on either side) for at most 2 * 16 * 2^-24 / 2^-9 = 2^-10 of the elements;
    # the terms' magnitudes may be up to 4 times r: 2^-8
    rng = np.random.default_rng([T, D])
    a = _inputs(rng, T, D, "bf16", yt, "f32", gates, True, True)
    r, h, _ = _check_forward(moe, a, "bf16", "f32")
    x, z = _terms(a)
    want = torch.from_numpy((x + z).astype(np.float32)).to(torch.bfloat16)
    assert (r.cpu() != want).double().mean() <= 2.0**-8
    R = _f64(r)
    ref = R * _rstd(R, True) * _f64(a["pre_weight"])
    assert (np.abs(_f64(h) - ref) <= (E + 2.0**-24) * np.abs(ref) + 1e-37).all()


def test_long_gate_groups(moe):
    # gate rows of many chunks each, a long sum over rows
    for T, D, gates in ((20000, 64, 2), (9000, 512, 3), (4099, 136, 1), (6000, 32, 3000)):
        print(f"norm long T={T} D={D} gates={gates}", flush=True)
        rng = np.random.default_rng(T)
        a = _inputs(rng, T, D, "f32", "f32", "f32", gates, True, True)
        r, h, stats = _check_forward(moe, a, "f32", "f32")
        _check_grad(moe, a, r, stats, _make(rng, (T, D), "f32"), _make(rng, (T, D), "f32"), "f32", "f32")


def test_against_differences(moe):
    # directional derivatives of a scalar of (r, h) in float64
    rng = np.random.default_rng(4)
    T, D = 6, 40
    a = _inputs(rng, T, D, "f32", "f32", "f32", 2, True, True)
    dr, dh = _make(rng, (T, D), "f32"), _make(rng, (T, D), "f32")
    r, h, stats = _check_forward(moe, a, "f32", "f32")
    grads = _check_grad(moe, a, r, stats, dr, dh, "f32", "f32")

    def value(v):
        y = v["y"] * _rstd(v["y"], True) * v["post_weight"] * np.repeat(v["gate"], 3, axis=0)
        R = ALPHA * v["x"] + BETA * y
        return (R * _f64(dr)).sum() + (R * _rstd(R, True) * v["pre_weight"] * _f64(dh)).sum()

    base = {k: _f64(t) for k, t in a.items()}
    for name, g in zip(("x", "y", "gate", "post_weight", "pre_weight"), grads):
        for _ in range(3):
            d = rng.standard_normal(base[name].shape)
            step = 1e-5
            up, down = ({**base, name: base[name] + s * step * d} for s in (1, -1))
            slope = (value(up) - value(down)) / (2 * step)
            scale = np.abs(_f64(g) * d).sum()
            # differences: step^2 of the third derivative and 2^-52 / step of the value;
            # the fp32 gradient: 4 E
            assert abs((_f64(g) * d).sum() - slope) <= (4 * E + 1e-7) * scale + 1e-7, name


def test_special_values_and_in_place(moe):
    rng = np.random.default_rng(6)
    a = _inputs(rng, 8, 64, "f32", "f32", "f32", 0, True, True)
    a["y"][1], a["x"][2] = 0, 0
    a["y"][2] = 0
    a["y"][3, 5] = float("inf")
    a["x"][4, 0] = float("nan")
    r, h, _ = moe.block_norm(a["x"], a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"])
    fin = torch.isfinite(r).all(dim=1).cpu().numpy()
    assert fin[[0, 1, 2, 5, 6, 7]].all() and not fin[3] and not fin[4]
    assert torch.equal(r[1], a["x"][1]) and (h[2] == 0).all()  # a zero row stays zero
    # r in the memory of x
    from mixtureofexperts_amd import _lib

    x = a["x"].clone()
    hh = torch.empty_like(x)
    _lib.check(_lib.lib().moe_block_norm_async(
        x.data_ptr(), 0, a["y"].data_ptr(), 0, a["post_weight"].data_ptr(), a["pre_weight"].data_ptr(), 0, None, 0, 0, 1.0,
        1.0, 1e-5, 8, 64, x.data_ptr(), hh.data_ptr(), 0, None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(x[[0, 1, 2, 5]], r[[0, 1, 2, 5]]) and torch.equal(hh[[0, 1, 2, 5]], h[[0, 1, 2, 5]])
    # a first norm: r is x
    r, h, _ = moe.block_norm(a["x"], pre_weight=a["pre_weight"])
    assert r is a["x"] and torch.isfinite(h[0]).all()


def test_no_rows(moe):
    w = torch.ones(32, device="cuda")
    x = torch.empty(0, 32, device="cuda")
    r, h, stats = moe.block_norm(x, x, pre_weight=w, post_weight=w)
    assert r.shape == h.shape == (0, 32) and stats.shape == (0, 2)
    dx, dy, dgate, dpost, dpre = moe.block_norm_grad(x, x, r, x, stats, pre_weight=w, post_weight=w)
    assert dx.shape == dy.shape == (0, 32) and dgate is None and (dpost == 0).all() and (dpre == 0).all()


def test_unaligned_rows(moe):
    # a view two elements into its buffer: 16-byte vectors do not fit
    rng = np.random.default_rng(12)
    a = _inputs(rng, 9, 128, "bf16", "bf16", "f32", 1, True, True)
    want = moe.block_norm(a["x"], a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"], gate=a["gate"])
    flat = torch.empty(9 * 128 + 2, dtype=torch.bfloat16, device="cuda")
    flat[2:] = a["x"].reshape(-1)
    got = moe.block_norm(flat[2:].view(9, 128), a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"],
                         gate=a["gate"])
    assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_graph_replay(moe):
    rng = np.random.default_rng(13)
    T, D = 300, 512
    sets = [_inputs(rng, T, D, "bf16", "f32", "f32", 3, True, True) for _ in range(3)]
    dr, dh = _make(rng, (T, D), "bf16"), _make(rng, (T, D), "bf16")

    def step(a):
        kw = dict(pre_weight=a["pre_weight"], post_weight=a["post_weight"], gate=a["gate"], alpha=ALPHA, beta=BETA)
        r, h, stats = moe.block_norm(a["x"], a["y"], **kw)
        return (r, h) + moe.block_norm_grad(dr, dh, r, a["y"], stats, **kw)

    want = [step(a) for a in sets]
    buf = {k: v.clone() for k, v in sets[0].items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for i in (0, 2, 1, 2):
        for k, v in sets[i].items():
            buf[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want[i])), i


@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 32)])
def test_no_rows_with_a_gate(moe, shape):
    # the sum over no rows is zero, also where the allocator's free blocks hold NaN
    print(f"norm no rows, gate {shape}", flush=True)
    w, gate = torch.ones(32, device="cuda"), torch.ones(shape, device="cuda")
    x = torch.empty(0, 32, device="cuda")
    _, _, stats = moe.block_norm(x, x, pre_weight=w, post_weight=w, gate=gate)
    for pre, post in itertools.product((w, None), (w, None)):
        dirt = [torch.full(s, float("nan"), device="cuda") for s in ((32,), (3, 32)) for _ in range(64)]
        del dirt
        dx, dy, dgate, dpost, dpre = moe.block_norm_grad(x, x if pre is not None else None, x, x, stats, pre_weight=pre,
                                                         post_weight=post, gate=gate)
        assert dx.shape == dy.shape == (0, 32) and dgate.shape == gate.shape
        for g in (dgate, dpost, dpre):
            assert g is None or (g == 0).all()


@pytest.mark.parametrize("T,D,yt,post,gates", [(2000, 4096, "f32", True, 2000), (3000, 328, "f32", False, 3), (700, 12000, "bf16", True, 0),
                                               (2500, 2050, "bf16", True, 1)])
def test_the_stream_does_not_depend_on_what_else_is_asked_for(moe, T, D, yt, post, gates):
    # r and rstd(y) with h in fp32, h in bf16 and no h, in the memory of x and not:
    # a forward pass computed again for its backward has to give the same bits.
    # (r formed once in fp64 and once in fp32 differs at one element in about 30000:
    # none in 980000 or more would be an accident of probability e^-30.)
    print(f"norm stream T={T} D={D} {yt} post={post} gates={gates}", flush=True)
    rng = np.random.default_rng([T, D, 3])
    a = _inputs(rng, T, D, "bf16", yt, "f32", gates, True, post)
    x, y, pre = a.pop("x"), a.pop("y"), a.pop("pre_weight")
    a.update(alpha=ALPHA, beta=BETA, eps=EPS)
    r, h32, stats = moe.block_norm(x, y, pre_weight=pre, h_dtype=torch.float32, **a)
    r16, h16, stats16 = moe.block_norm(x, y, pre_weight=pre, **a)
    r0, none, stats0 = moe.block_norm(x, y, **a)
    assert none is None and torch.equal(r, r16) and torch.equal(r, r0)
    assert torch.equal(stats, stats16) and torch.equal(stats[:, 0], stats0[:, 0])
    assert torch.equal(h16, h32.to(torch.bfloat16))


def test_bf16_stream_is_formed_closer_than_in_fp32(moe):
    # against the float64 formula's r, rounded by way of fp32 as torch does: r formed
    # in fp32 by plain operations lands on the other bf16 neighbour at about one
    # element in 30000 (250 of these), at most a third as often may the call; every
    # such r is one bf16 step off, so h's distance from the norm of the right r is
    # at most sqrt(1/3) of theirs, 0.7 with room for the sizes of the values hit
    T, D = 2000, 4096
    print("norm bf16 stream, fp64 against fp32", flush=True)
    rng = np.random.default_rng(77)
    a = _inputs(rng, T, D, "bf16", "f32", "f32", T, True, True)
    x, z = _terms(a)
    want = torch.from_numpy((x + z).astype(np.float32)).to(torch.bfloat16)
    r, h, _ = moe.block_norm(a["x"], a["y"], pre_weight=a["pre_weight"], post_weight=a["post_weight"], gate=a["gate"],
                             alpha=ALPHA, beta=BETA, eps=EPS, h_dtype=torch.float32)
    f = lambda t: t.float().cpu()
    y = f(a["y"])
    zf = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * f(a["post_weight"]) * f(a["gate"])
    plain = (ALPHA * f(a["x"]) + BETA * zf).to(torch.bfloat16)
    flips, fp32 = int((r.cpu() != want).sum()), int((plain != want).sum())
    print("other neighbour:", flips, "in fp32:", fp32, flush=True)
    assert fp32 >= 100 and 3 * flips <= fp32
    W = _f64(want)
    ref = W * _rstd(W, True) * _f64(a["pre_weight"])
    P = _f64(plain)
    off = np.linalg.norm(_f64(h) - ref) / np.linalg.norm(ref)
    off32 = np.linalg.norm(P * _rstd(P, True) * _f64(a["pre_weight"]) - ref) / np.linalg.norm(ref)
    assert off <= 0.7 * off32, (off, off32)


@pytest.mark.parametrize("T,D", [(2**21 + 5, 8), (2**22 + 2**20 + 3, 16), (2**20 + 7, 520)])
def test_millions_of_rows(moe, T, D):
    # more rows than one dimension of a launch takes; compared with the same rows in
    # parts, a part at the end in float64
    print(f"norm rows T={T} D={D}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T)
    new = lambda r: torch.randn(r, D, generator=g, device="cuda").to(torch.bfloat16)
    x, y, gate, pre = new(T), new(T), new(1), new(1)[0].float()
    kw = dict(pre_weight=pre, post_weight=pre, gate=gate, alpha=ALPHA, beta=BETA, eps=EPS)
    r, h, stats = moe.block_norm(x, y, **kw)
    cut = T // 2 // 4 * 4
    for s in (slice(0, cut), slice(cut, T)):
        for got, part in zip((r, h, stats), moe.block_norm(x[s], y[s], **kw)):
            assert torch.equal(got[s], part)
    tail = slice(T - 999, T)
    _check_forward(moe, dict(x=x[tail], y=y[tail], pre_weight=pre, post_weight=pre, gate=gate), "bf16", "bf16")
    dr, dh = new(T), new(T)
    dx, dy, dgate, dpost, dpre = moe.block_norm_grad(dr, dh, r, y, stats, **{k: v for k, v in kw.items() if k != "eps"})
    a = dict(x=x[tail], y=y[tail], pre_weight=pre, post_weight=pre, gate=gate)
    (wx, wy, *_), (mx, my, *_) = _formula(a, dr[tail], dh[tail], r[tail])
    for got, ref, mag in ((dx, wx, mx), (dy, wy, my)):
        assert (np.abs(_f64(got[tail]) - ref) <= 4 * E * mag + HALF["bf16"] * np.abs(ref) + 1e-37).all()
    # the column sums, in float64 on the GPU: a rounding of fp32 per addition, in
    # chunks of T / 512 rows at most, whose sums are added in turn
    rh = r.double() * stats[:, 1:].double()
    ref, mag = (dh.double() * rh).sum(0), (dh.double() * rh).abs().sum(0)
    assert ((dpre.double() - ref).abs() <= (T / 512 + 2048) * 2.0**-24 * mag).all()


@pytest.mark.parametrize("T,D", [(800, 1024), (300, 4100), (60, 16384), (900, 331)])
def test_gated_bf16_stream_to_the_bit(moe, T, D):
    # without a post norm the formula's fp64 value is exact (bf16 factors), so r has one
    # right answer, by way of fp32, also where the two terms cancel; and rows of zeros,
    # infinities, NaN and products past fp32's range on the way
    print(f"norm gated stream T={T} D={D}", flush=True)
    rng = np.random.default_rng([T, D, 5])
    y, gate = _make(rng, (T, D), "bf16"), _make(rng, (T, D), "bf16")
    z = -(BETA * y.double() * gate.double()) / ALPHA
    x = torch.where(torch.rand(T, D, device="cuda") < 0.5, z, torch.randn(T, D, device="cuda").double()).to(torch.bfloat16)
    x[3], y[3], gate[4] = 0, 0, 0
    x[5, 7], y[6, D - 1], gate[7, 0], y[8, 1] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[9, 2], y[9, 2] = float("inf"), float("inf")
    y[10], gate[10] = 2.0**120, 2.0**-120
    y[11], gate[11] = -(2.0**-130), 2.0**100
    want = (ALPHA * x.double() + BETA * (y.double() * gate.double())).float().to(torch.bfloat16)
    for pre, ht in ((None, None), (torch.ones(D, device="cuda"), torch.bfloat16), (torch.ones(D, device="cuda"), torch.float32)):
        r, h, stats = moe.block_norm(x, y, gate=gate, pre_weight=pre, alpha=ALPHA, beta=BETA, h_dtype=ht)
        bad = ~((r == want) | (torch.isnan(r) & torch.isnan(want)))
        assert not bad.any(), bad.nonzero()[:5]
    assert torch.isnan(want[5, 7]) and torch.isinf(want[6, D - 1]) and torch.isnan(want[9, 2]) == torch.isnan(r[9, 2])
