"""What quantize_fp8 and fp8_matmul refuse, at the C entry points and in Python.  Every
call here is refused on the host: the pointers are never read."""
import ctypes

import pytest

P = 0x10000  # an aligned address that no refused call reads
F32, BF16, FP8, INT8 = 0, 1, 2, 3

QUANT = dict(x=P, ldx=64, x_stride=640, x_dtype=BF16, matrices=2, rows=10, cols=64, block_rows=1, q=2 * P, ldq=64, q_stride=640,
             scale=3 * P, stream=None)
# 10 rows of 64 -> 32 in 4 groups; the rows quantised: 10 scales (48 bytes) and 10 x 64 codes
MM = dict(x=P, ldx=64, x_dtype=BF16, x_scale=None, w=2 * P, ldw=64, w_stride=64 * 32, w_scale=3 * P, offsets=4 * P, groups=4,
          rows=10, in_dim=64, out_dim=32, y=5 * P, ldy=32, y_dtype=BF16, workspace=6 * P, workspace_bytes=48 + 640, stream=None)


def _refused(fn, args, msg):
    from mixtureofexperts_amd import _lib

    rc = getattr(_lib.lib(), fn)(*args.values())
    text = _lib.lib().moe_last_error(None).decode()
    assert rc == _lib.MOE_EINVAL, (rc, args)
    assert fn in text and msg in text, text


@pytest.mark.parametrize("bad,msg", [
    (dict(x_dtype=INT8), "x_dtype"), (dict(x_dtype=FP8), "x_dtype"), (dict(block_rows=0), "block_rows"),
    (dict(block_rows=64), "block_rows"), (dict(rows=-1), "rows"), (dict(matrices=-1), "matrices"), (dict(cols=0), "cols"),
    (dict(rows=2**30 + 1), "2^30"), (dict(cols=2**30 + 1, ldx=2**31, ldq=2**31), "2^30"), (dict(ldx=63), "row stride"),
    (dict(ldq=63), "row stride"), (dict(x_stride=639), "matrix stride"), (dict(q_stride=639), "matrix stride"),
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(x=P + 1), "aligned"),
    (dict(scale=3 * P + 2), "aligned"), (dict(q=P + 2 * 1280 - 1), "overlap"), (dict(q=P - 1279), "overlap"),
    (dict(scale=P + 1276), "overlap"), (dict(scale=2 * P + 1276), "overlap"), (dict(scale=2 * P - 76), "overlap"),
])
def test_quantize_refuses(moe, bad, msg):
    _refused("moe_quantize_fp8_async", {**QUANT, **bad}, msg)


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "groups"), (dict(rows=-1), "rows"), (dict(in_dim=0), "dimensions"), (dict(offsets=None), "offsets"),
    (dict(rows=2**30 + 1), "2^30"), (dict(x_dtype=INT8), "x_dtype"), (dict(y_dtype=FP8), "result"), (dict(ldx=63), "row stride"),
    (dict(ldw=63), "row stride"), (dict(ldy=31), "row stride"), (dict(w_stride=64 * 32 - 1), "w_stride"),
    (dict(w_scale=None), "null"), (dict(y=None), "null"), (dict(x_dtype=FP8), "x_scale"), (dict(workspace=None), "workspace"),
    (dict(workspace=6 * P + 8), "workspace"), (dict(workspace_bytes=48 + 639), "workspace"), (dict(x=P + 1), "aligned"),
    (dict(w_scale=3 * P + 2), "aligned"), (dict(x_dtype=FP8, x_scale=7 * P + 2), "aligned"), (dict(y=P), "overlap"),
    (dict(y=2 * P + 4 * 64 * 32 - 2), "overlap"), (dict(y=3 * P + 12), "overlap"), (dict(y=4 * P + 16), "overlap"),
    (dict(x_dtype=FP8, x_scale=7 * P, y=7 * P + 36), "overlap"),
])
def test_matmul_refuses(moe, bad, msg):
    _refused("moe_fp8_matmul_async", {**MM, **bad}, msg)


def test_workspaces(moe):
    from mixtureofexperts_amd import _lib

    L, n = _lib.lib(), ctypes.c_int64(-1)
    assert L.moe_fp8_matmul_workspace(4, 10, 64, 32, BF16, ctypes.byref(n)) == 0 and n.value == 48 + 640
    assert L.moe_fp8_matmul_workspace(4, 10, 64, 32, FP8, ctypes.byref(n)) == 0 and n.value == 0
    assert L.moe_fp8_matmul_workspace(1, 3, 100000, 48, FP8, ctypes.byref(n)) == 0 and n.value > 0
    assert L.moe_fp8_matmul_workspace(8, 0, 64, 32, BF16, ctypes.byref(n)) == 0 and n.value == 0
    assert L.moe_fp8_matmul_workspace(8, 2**30, 64, 32, BF16, ctypes.byref(n)) == 0 and n.value >= 68 * 2**30
    assert L.moe_fp8_matmul_workspace(0, 3, 8, 8, FP8, ctypes.byref(n)) == _lib.MOE_EINVAL
    assert L.moe_fp8_matmul_workspace(1, 3, 8, 8, FP8, None) == _lib.MOE_EINVAL


def test_empty_calls_are_no_work(moe):
    from mixtureofexperts_amd import _lib

    L = _lib.lib()
    assert L.moe_quantize_fp8_async(*{**QUANT, "rows": 0, "x": None}.values()) == 0
    assert L.moe_quantize_fp8_async(*{**QUANT, "matrices": 0, "x": None}.values()) == 0
    assert L.moe_fp8_matmul_async(*{**MM, "rows": 0, "workspace": None, "x": None}.values()) == 0


def test_more_tiles_than_a_launch_are_refused(moe):
    _refused("moe_fp8_matmul_async",
             {**MM, "x": 2**44, "w": 2**45, "offsets": 2**46, "y": 2**56, "rows": 2**30, "out_dim": 2**20, "ldy": 2**20,
              "w_stride": 2**26, "x_dtype": FP8, "x_scale": 2**43, "w_scale": 2**42}, "too many tiles")


def _calls(moe, mark, dev):
    torch = pytest.importorskip("torch")
    z = lambda *s: torch.zeros(*s, device=dev)
    f8 = lambda *s: torch.zeros(*s, device=dev, dtype=torch.float8_e4m3fn)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    w, ws = (2, 6, 8), (2, 1, 1)
    return [
        ("x", lambda: moe.quantize_fp8(mark(z(4, 8)))),
        ("x", lambda: moe.quantize_fp8(mark(z(4, 8)), block_rows=128)),
        ("x", lambda: moe.fp8_matmul(mark(z(4, 8)), f8(*w), z(*ws), off)),
        ("w_scale", lambda: moe.fp8_matmul(z(4, 8), f8(*w), mark(z(*ws)), off)),
        ("x_scale", lambda: moe.fp8_matmul(f8(4, 8), f8(*w), z(*ws), off, x_scale=mark(z(4, 1)))),
        ("out", lambda: moe.fp8_matmul(z(4, 8), f8(*w), z(*ws), off, out=mark(z(4, 6)))),
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
    torch = pytest.importorskip("torch")
    with pytest.raises(moe.MoeError, match="block_rows"):
        moe.quantize_fp8(torch.zeros(4, 8), block_rows=32)


@pytest.mark.gpu
def test_python_refuses(moe):
    torch = pytest.importorskip("torch")
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")
    f8, e5 = torch.float8_e4m3fn, torch.float8_e5m2
    x, w, ws, off = z(4, 200), z(2, 130, 200, t=f8), z(2, 2, 2), z(3, t=torch.int32)
    calls = [
        (lambda: moe.quantize_fp8(x.half()), "must be"),
        (lambda: moe.quantize_fp8(z(3, 2, 0)), "columns"),
        (lambda: moe.quantize_fp8(z(4), block_rows=128), "dimensions"),
        (lambda: moe.quantize_fp8(z(2, 2, 4, 8), block_rows=128), "dimensions"),
        (lambda: moe.quantize_fp8(x.t()), "contiguous"),
        (lambda: moe.quantize_fp8(z(1, 4, 8).expand(2, 4, 8), block_rows=128), "overlap"),
        (lambda: moe.fp8_matmul(x.half(), w, ws, off), "must be"),
        (lambda: moe.fp8_matmul(x, w.view(torch.uint8), ws, off), "must be"),
        (lambda: moe.fp8_matmul(x, w.view(e5), ws, off), "must be"),
        (lambda: moe.fp8_matmul(x, w, ws[:, :1], off), "w_scale"),
        (lambda: moe.fp8_matmul(x, w, ws.transpose(1, 2), off), "w_scale"),
        (lambda: moe.fp8_matmul(x, w, ws), "offsets are needed"),
        (lambda: moe.fp8_matmul(x[:, :199], w, ws, off), "columns"),
        (lambda: moe.fp8_matmul(z(4, 200, t=f8), w, ws, off), "x_scale"),
        (lambda: moe.fp8_matmul(z(4, 200, t=f8), w, ws, off, x_scale=z(4, 1)), "x_scale"),
        (lambda: moe.fp8_matmul(x, w, ws, off, x_scale=z(4, 2)), "x_scale"),
        (lambda: moe.fp8_matmul(x, w, ws, off, out_dtype=torch.int8), "result must be"),
        (lambda: moe.fp8_matmul(x, w, ws, off, out=z(4, 129)), "out must be"),
        (lambda: moe.fp8_matmul(x, w, ws, off, out=x[:, :130]), "overlap"),
        (lambda: moe.fp8_matmul(x, w, ws, off.cpu()), "one device"),
    ]
    for i, (call, msg) in enumerate(calls):
        with pytest.raises(moe.MoeError, match=msg):
            call()
            print("not refused:", i, flush=True)
