"""What gated_matmul and its gradients refuse, at the C entry points and in Python.
Every call here is refused on the host: the pointers are never read."""
import ctypes

import pytest

P = 0x10000  # an aligned address that no refused call reads
F32, BF16, FP8, INT8 = 0, 1, 2, 3
FLUX, LLAMA = 0, 1
GELU, SILU = 0, 1

# distinct places, 4 groups of 64 -> 32 over 10 rows
WS = dict(workspace=None, workspace_bytes=0, stream=None)
FORWARD = dict(x=P, ldx=64, w1=2 * P, ldw1=64, w1_stride=64 * 32, w3=3 * P, ldw3=64, w3_stride=64 * 32, layout=LLAMA,
               activation=SILU, offsets=4 * P, groups=4, rows=10, in_dim=64, hidden_dim=32, dtype=BF16, h=5 * P, ldh=32,
               h_dtype=BF16, a=6 * P, lda=32, b=7 * P, ldb=32, **WS)
GRAD = dict(dy=P, lddy=64, w2=2 * P, ldw2=32, w2_stride=64 * 32, layout=LLAMA, activation=SILU, a=3 * P, lda=32, b=4 * P,
            ldb=32, offsets=5 * P, groups=4, rows=10, hidden_dim=32, out_dim=64, dtype=BF16, da=6 * P, ldda=32, db=7 * P,
            lddb=32, h=8 * P, ldh=32, **WS)
GRADX = dict(da=P, ldda=32, db=2 * P, lddb=32, w1=3 * P, ldw1=64, w1_stride=64 * 32, w3=4 * P, ldw3=64, w3_stride=64 * 32,
             layout=LLAMA, offsets=5 * P, groups=4, rows=10, in_dim=64, hidden_dim=32, dtype=BF16, dx=6 * P, lddx=64,
             dx_dtype=BF16, **WS)


def _refused(fn, args, msg):
    from mixtureofexperts_amd import _lib

    rc = getattr(_lib.lib(), fn)(*args.values())
    text = _lib.lib().moe_last_error(None).decode()
    assert rc == _lib.MOE_EINVAL, (rc, args)
    assert fn in text and msg in text, text


COMMON = [(dict(groups=0), "groups"), (dict(rows=-1), "rows"), (dict(offsets=None), "offsets"), (dict(dtype=FP8), "dtype"),
          (dict(layout=2), "layout"), (dict(rows=2**30 + 1), "2^30"), (dict(groups=2**30 + 1), "2^30"),
          (dict(hidden_dim=0), "dimensions")]


@pytest.mark.parametrize("bad,msg", COMMON + [
    (dict(in_dim=0), "dimensions"), (dict(activation=4), "activation"), (dict(activation=-1), "activation"),
    (dict(dtype=F32), "fp32"), (dict(h_dtype=INT8), "result"), (dict(a=None), "come together"), (dict(b=None), "come together"),
    (dict(ldx=63), "row stride"), (dict(ldw1=63), "row stride"), (dict(ldw3=63), "row stride"), (dict(ldh=31), "row stride"),
    (dict(lda=31), "row stride"), (dict(ldb=31), "row stride"), (dict(w1_stride=64 * 32 - 1), "stride"),
    (dict(w3_stride=64 * 32 - 1), "stride"), (dict(x=None), "null"), (dict(w1=None), "null"), (dict(w3=None), "null"),
    (dict(h=None), "null"), (dict(x=P + 1), "aligned"), (dict(w3=3 * P + 1), "aligned"), (dict(b=7 * P + 1), "aligned"),
    (dict(h=5 * P + 2, h_dtype=F32), "aligned"),
])
def test_forward_refuses(moe, bad, msg):
    _refused("moe_gated_matmul_async", {**FORWARD, **bad}, msg)


@pytest.mark.parametrize("bad,msg", COMMON + [
    (dict(out_dim=0), "dimensions"), (dict(activation=9), "activation"), (dict(lddy=63), "row stride"),
    (dict(ldw2=31), "row stride"), (dict(lda=31), "row stride"), (dict(ldb=31), "row stride"), (dict(ldda=31), "row stride"),
    (dict(lddb=31), "row stride"), (dict(ldh=31), "row stride"), (dict(w2_stride=64 * 32 - 1), "w2_stride"),
    (dict(w2=None), "out_dim must be"), (dict(dy=None), "null"), (dict(a=None), "null"), (dict(db=None), "null"),
    (dict(h=None), "null"), (dict(da=6 * P + 1), "aligned"), (dict(w2=2 * P + 1), "aligned"),
])
def test_gradient_refuses(moe, bad, msg):
    _refused("moe_gated_matmul_grad_async", {**GRAD, **bad}, msg)


@pytest.mark.parametrize("bad,msg", COMMON + [
    (dict(in_dim=0), "dimensions"), (dict(ldda=31), "row stride"), (dict(lddb=31), "row stride"), (dict(lddx=63), "row stride"),
    (dict(ldw3=63), "row stride"), (dict(w3_stride=64 * 32 - 1), "stride"), (dict(db=None), "null"), (dict(dx=None), "null"),
    (dict(dx=6 * P + 2, dx_dtype=F32), "aligned"), (dict(dtype=F32), "fp32"),
])
def test_row_gradient_refuses(moe, bad, msg):
    _refused("moe_gated_matmul_grad_x_async", {**GRADX, **bad}, msg)


def test_results_on_operands_or_each_other_are_refused(moe):
    for name in ("h", "a", "b"):
        for at in (P, P + 9 * 128 + 126, 2 * P + 2 * 4 * 64 * 32 - 2, 3 * P, 4 * P + 16):
            _refused("moe_gated_matmul_async", {**FORWARD, name: at}, "overlap")
    for one, two in (("h", "a"), ("h", "b"), ("a", "b")):
        _refused("moe_gated_matmul_async", {**FORWARD, one: FORWARD[two] + 10 * 64 - 2}, "overlap each other")
    for name in ("da", "db", "h"):
        for at in (P, 2 * P, 3 * P, 4 * P, 5 * P + 16):
            _refused("moe_gated_matmul_grad_async", {**GRAD, name: at}, "overlap")
    _refused("moe_gated_matmul_grad_async", {**GRAD, "w2": None, "out_dim": 32, "lddy": 32, "da": P + 2}, "overlap")
    _refused("moe_gated_matmul_grad_async", {**GRAD, "db": 6 * P}, "overlap each other")
    for at in (P, 2 * P, 3 * P, 4 * P, 5 * P + 16):
        _refused("moe_gated_matmul_grad_x_async", {**GRADX, "dx": at}, "overlap")


def test_workspaces(moe):
    from mixtureofexperts_amd import _lib

    L, n = _lib.lib(), ctypes.c_int64(-1)
    far = dict(offsets=None, groups=1, rows=3)
    big = 2**40
    for fn, sizes, args in (
            ("moe_gated_matmul", (1, 3, 100000, 48),
             {**FORWARD, **far, "in_dim": 100000, "hidden_dim": 48, "ldx": 100000, "ldw1": 100000, "ldw3": 100000, "ldh": 48,
              "lda": 48, "ldb": 48, "h": big, "a": 2 * big, "b": 3 * big}),
            ("moe_gated_matmul_grad", (1, 3, 48, 100000),
             {**GRAD, **far, "out_dim": 100000, "hidden_dim": 48, "lddy": 100000, "ldw2": 48, "lda": 48, "ldb": 48, "ldda": 48,
              "lddb": 48, "ldh": 48, "da": big, "db": 2 * big, "h": 3 * big}),
            ("moe_gated_matmul_grad_x", (1, 3, 48, 100000),
             {**GRADX, **far, "in_dim": 48, "hidden_dim": 100000, "ldda": 100000, "lddb": 100000, "ldw1": 48, "ldw3": 48,
              "lddx": 48, "dx": big})):
        query = getattr(L, fn + "_workspace")
        assert query(*sizes, BF16, ctypes.byref(n)) == 0 and n.value > 0, fn
        for ws, size in ((None, n.value), (P + 8, n.value), (P, 16)):
            _refused(fn + "_async", {**args, "workspace": ws, "workspace_bytes": size}, "workspace")
        assert query(8, 0, 64, 32, BF16, ctypes.byref(n)) == 0 and n.value == 0
        # (the row gradient splits the last round of few large tiles)
        assert query(8, 8192, 4096, 14336, BF16, ctypes.byref(n)) == 0 and (n.value > 0) == (fn == "moe_gated_matmul_grad_x")
        assert query(8, 8192, 4096, 14336, F32, ctypes.byref(n)) == 0 and n.value == 0
        assert query(1, 3, 8, 8, FP8, ctypes.byref(n)) == _lib.MOE_EINVAL
        assert query(1, 3, 8, 8, BF16, None) == _lib.MOE_EINVAL
        assert query(0, 3, 8, 8, BF16, ctypes.byref(n)) == _lib.MOE_EINVAL


def test_empty_calls_are_no_work(moe):
    from mixtureofexperts_amd import _lib

    L = _lib.lib()
    assert L.moe_gated_matmul_async(*{**FORWARD, "rows": 0, "x": None, "h": None}.values()) == 0
    assert L.moe_gated_matmul_grad_async(*{**GRAD, "rows": 0, "dy": None}.values()) == 0
    assert L.moe_gated_matmul_grad_x_async(*{**GRADX, "rows": 0, "dx": None}.values()) == 0


def test_more_tiles_than_a_launch_are_refused(moe):
    far = dict(x=2**44, w1=2**45, w3=2**46, offsets=2**47, h=2**56, a=None, b=None)
    _refused("moe_gated_matmul_async", {**FORWARD, **far, "rows": 2**30, "hidden_dim": 2**20, "ldh": 2**20, "w1_stride": 2**26,
                                        "w3_stride": 2**26}, "too many tiles")


def _calls(moe, mark, dev):
    torch = pytest.importorskip("torch")
    z = lambda *s: torch.zeros(*s, device=dev)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    w, w2 = (2, 6, 8), (2, 8, 6)
    outs = lambda i, n: tuple(mark(z(4, n)) if k == i else z(4, n) for k in range(3))
    return [
        ("x", lambda: moe.gated_matmul(mark(z(4, 8)), z(*w), z(*w), off)),
        ("w1", lambda: moe.gated_matmul(z(4, 8), mark(z(*w)), z(*w), off)),
        ("w3", lambda: moe.gated_matmul(z(4, 8), z(*w), mark(z(*w)), off)),
        ("out", lambda: moe.gated_matmul(z(4, 8), z(*w), z(*w), off, out=mark(z(4, 6)))),
        ("out", lambda: moe.gated_matmul(z(4, 8), z(*w), z(*w), off, save=True, out=outs(2, 6))),
        ("dy", lambda: moe.gated_matmul_grad(mark(z(4, 8)), z(4, 6), z(4, 6), z(*w2), off)),
        ("a", lambda: moe.gated_matmul_grad(z(4, 8), mark(z(4, 6)), z(4, 6), z(*w2), off)),
        ("b", lambda: moe.gated_matmul_grad(z(4, 8), z(4, 6), mark(z(4, 6)), z(*w2), off)),
        ("w2", lambda: moe.gated_matmul_grad(z(4, 8), z(4, 6), z(4, 6), mark(z(*w2)), off)),
        ("out", lambda: moe.gated_matmul_grad(z(4, 6), z(4, 6), z(4, 6), None, off, out=outs(1, 6))),
        ("da", lambda: moe.gated_matmul_grad_x(mark(z(4, 6)), z(4, 6), z(*w), z(*w), off)),
        ("db", lambda: moe.gated_matmul_grad_x(z(4, 6), mark(z(4, 6)), z(*w), z(*w), off)),
        ("w1", lambda: moe.gated_matmul_grad_x(z(4, 6), z(4, 6), mark(z(*w)), z(*w), off)),
        ("out", lambda: moe.gated_matmul_grad_x(z(4, 6), z(4, 6), z(*w), z(*w), off, out=mark(z(4, 8)))),
    ]


def test_what_autograd_would_record_is_refused(moe):
    torch = pytest.importorskip("torch")
    fwd = torch.autograd.forward_ad
    for name, call in _calls(moe, lambda t: t.requires_grad_(), "cpu"):
        with pytest.raises(moe.MoeError, match=f"{name} requires a gradient"):
            call()
    with fwd.dual_level():
        for name, call in _calls(moe, lambda t: fwd.make_dual(t, torch.ones_like(t)), "cpu"):
            with pytest.raises(moe.MoeError, match=f"{name} carries a tangent"):
                call()


def test_host_tensors_are_refused(moe):
    for _, call in _calls(moe, lambda t: t, "cpu"):
        with pytest.raises(moe.MoeError, match="GPU memory"):
            call()


@pytest.mark.gpu
def test_python_refuses(moe):
    torch = pytest.importorskip("torch")
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")
    x, w, w2, off, g = z(4, 8), z(2, 6, 8), z(2, 8, 6), z(3, t=torch.int32), z(4, 6)
    calls = [
        (lambda: moe.gated_matmul(x.half(), w, w, off), "must be"),
        (lambda: moe.gated_matmul(x, w.float(), w, off), "must be"),
        (lambda: moe.gated_matmul(x, w, w[:, :5], off), "one shape"),
        (lambda: moe.gated_matmul(x, w, w), "offsets are needed"),
        (lambda: moe.gated_matmul(x[:, :7], w, w, off), "columns"),
        (lambda: moe.gated_matmul(x, w, w, off, activation=torch.tanh), "activation"),
        (lambda: moe.gated_matmul(x, w, w, off, layout=3), "layout"),
        (lambda: moe.gated_matmul(x, w, w, off, out=z(4, 7)), "out must be"),
        (lambda: moe.gated_matmul(x, w, w, off, save=True, out=z(4, 6)), "out must be"),
        (lambda: moe.gated_matmul(x, w, w, off, save=True, out=(g, g, z(4, 7))), "b must be"),
        (lambda: moe.gated_matmul(x, w, w, off, save=True, out=(g, z(4, 6), z(4, 6, t=torch.float32))), "b must be"),
        (lambda: moe.gated_matmul(x, w, w, off, save=True, out=(g, g, z(4, 6))), "overlap"),
        (lambda: moe.gated_matmul(x, w, w, off, out_dtype=torch.int8), "result must be"),
        (lambda: moe.gated_matmul(x, w, w, off.cpu()), "one device"),
        (lambda: moe.gated_matmul(z(1, 8).expand(4, 8), w, w, off), "overlap"),
        (lambda: moe.gated_matmul_grad(x, g, g[:3], w2, off), "one shape"),
        (lambda: moe.gated_matmul_grad(x, g, g, w2[:, :, :5], off), "w2 takes"),
        (lambda: moe.gated_matmul_grad(x[:, :7], g, g, w2, off), "columns"),
        (lambda: moe.gated_matmul_grad(x, g, g, None, off), "columns"),
        (lambda: moe.gated_matmul_grad(x, g.float(), g, w2, off), "must be"),
        (lambda: moe.gated_matmul_grad(g, g, g, None, off[:1]), "two row numbers"),
        (lambda: moe.gated_matmul_grad(g, g, g, None, off, out=(z(4, 6), g, z(4, 6))), "overlap"),
        (lambda: moe.gated_matmul_grad_x(g, g[:3], w, w, off), "one shape"),
        (lambda: moe.gated_matmul_grad_x(x, x, w, w, off), "columns"),
        (lambda: moe.gated_matmul_grad_x(g, g, w, w, off, out=x[:, :7]), "out must be"),
    ]
    for i, (call, msg) in enumerate(calls):
        with pytest.raises(moe.MoeError, match=msg):
            call()
            print("not refused:", i, flush=True)
