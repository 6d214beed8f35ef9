"""What the operators on device tensors refuse, at the C entry points and in
the Python functions.  Every call here is refused on the host: the pointers
are never read."""
import ctypes

import pytest

P = 0x10000  # an aligned address that no refused call reads
F32, BF16, FP8, INT8 = 0, 1, 2, 3
FLUX, LLAMA = 0, 1

ROWS = dict(x=P, ldx=64, w=P, ldw=64, w_stride=64 * 32, layout=LLAMA, offsets=P, groups=4, rows=10, in_dim=64, out_dim=32,
            dtype=BF16, y=P, ldy=32, y_dtype=BF16, workspace=None, workspace_bytes=0, stream=None)


def _refused(moe, fn, args, msg):
    from mixtureofexperts_amd import _lib

    rc = getattr(_lib.lib(), fn)(*args.values())
    text = _lib.lib().moe_last_error(None).decode()
    assert rc == _lib.MOE_EINVAL, (rc, args)
    assert fn in text and msg in text, text


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "groups"), (dict(rows=-1), "rows"), (dict(in_dim=0), "dimensions"), (dict(out_dim=-3), "dimensions"),
    (dict(offsets=None), "offsets"), (dict(dtype=FP8), "dtype"), (dict(dtype=7), "dtype"), (dict(y_dtype=FP8), "result"),
    (dict(dtype=F32, y_dtype=BF16), "fp32"), (dict(layout=2), "layout"), (dict(ldx=63), "row stride"),
    (dict(ldy=31), "row stride"), (dict(ldw=63), "row stride"), (dict(w_stride=64 * 31), "w_stride"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(x=P + 1), "aligned"),
    (dict(w=P + 1), "aligned"), (dict(y=P + 1), "aligned"), (dict(y=P + 2, y_dtype=F32), "aligned"),
])
def test_grouped_matmul_refuses(moe, bad, msg):
    _refused(moe, "moe_grouped_matmul_async", {**ROWS, **bad}, msg)


@pytest.mark.parametrize("bad,msg", [(dict(ldx=31), "row stride"), (dict(ldy=63), "row stride"), (dict(dtype=FP8), "dtype"),
                                     (dict(y=None), "null"), (dict(offsets=None), "offsets")])
def test_grouped_matmul_grad_x_refuses(moe, bad, msg):
    _refused(moe, "moe_grouped_matmul_grad_x_async", {**ROWS, "ldx": 32, "ldy": 64, **bad}, msg)


GRADW = dict(x=P, ldx=64, dy=P, lddy=32, layout=LLAMA, offsets=P, groups=4, rows=10, in_dim=64, out_dim=32, dtype=BF16,
             dw=P, lddw=64, dw_stride=64 * 32, dw_dtype=F32, accumulate=0, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "groups"), (dict(rows=-1), "rows"), (dict(offsets=None), "offsets"), (dict(dtype=INT8), "dtype"),
    (dict(dtype=F32, dw_dtype=BF16), "fp32"), (dict(layout=-1), "layout"), (dict(ldx=63), "row stride"),
    (dict(lddy=31), "row stride"), (dict(lddw=63), "row stride"), (dict(dw_stride=64 * 31), "dw_stride"),
    (dict(x=None), "null"), (dict(dw=None), "null"), (dict(dw=P + 2), "aligned"), (dict(dy=P + 1), "aligned"),
])
def test_grouped_matmul_grad_w_refuses(moe, bad, msg):
    _refused(moe, "moe_grouped_matmul_grad_w_async", {**GRADW, **bad}, msg)


def test_grad_w_refuses_a_small_workspace(moe):
    from mixtureofexperts_amd import _lib

    L, n = _lib.lib(), ctypes.c_int64(-1)
    # one group of many rows and a small matrix: its rows may be split over workgroups
    assert L.moe_grouped_matmul_grad_w_workspace(1, 100000, 64, 64, ctypes.byref(n)) == 0 and n.value >= 0
    if n.value:
        args = {**GRADW, "groups": 1, "rows": 100000, "out_dim": 64, "lddy": 64, "lddw": 64}
        for ws, size in ((None, n.value), (P, n.value - 1), (P + 8, n.value)):
            _refused(moe, "moe_grouped_matmul_grad_w_async", {**args, "workspace": ws, "workspace_bytes": size},
                     "workspace")
    assert L.moe_grouped_matmul_grad_w_workspace(0, 1, 1, 1, ctypes.byref(n)) == _lib.MOE_EINVAL
    assert L.moe_grouped_matmul_grad_w_workspace(1, 1, 1, 1, None) == _lib.MOE_EINVAL


def test_matmul_refuses_a_small_workspace(moe):
    from mixtureofexperts_amd import _lib

    L, n = _lib.lib(), ctypes.c_int64(-1)
    # three rows against a narrow matrix: the long sum is split over workgroups
    assert L.moe_grouped_matmul_workspace(1, 3, 100000, 48, BF16, ctypes.byref(n)) == 0 and n.value > 0
    args = {**ROWS, "groups": 1, "rows": 3, "in_dim": 100000, "out_dim": 48, "ldx": 100000, "ldw": 100000, "ldy": 48}
    for ws, size in ((None, n.value), (P + 8, n.value), (P, 16)):
        _refused(moe, "moe_grouped_matmul_async", {**args, "workspace": ws, "workspace_bytes": size}, "workspace")
    assert L.moe_grouped_matmul_workspace(8, 8192, 4096, 14336, BF16, ctypes.byref(n)) == 0 and n.value == 0
    assert L.moe_grouped_matmul_workspace(1, 3, 8, 8, FP8, ctypes.byref(n)) == _lib.MOE_EINVAL
    assert L.moe_grouped_matmul_workspace(1, 3, 8, 8, BF16, None) == _lib.MOE_EINVAL
    assert L.moe_int8_matmul_workspace(1, 3, 100000, 48, INT8, ctypes.byref(n)) == 0 and n.value > 0
    assert L.moe_int8_matmul_workspace(0, 3, 8, 8, INT8, ctypes.byref(n)) == _lib.MOE_EINVAL


QUANT = dict(x=P, ldx=64, x_dtype=BF16, rows=4, cols=64, q=P, ldq=64, scale=P, stream=None)


@pytest.mark.parametrize("bad,msg", [
    (dict(x_dtype=INT8), "x_dtype"), (dict(rows=-1), "rows"), (dict(cols=0), "cols"), (dict(ldx=63), "row stride"),
    (dict(ldq=63), "row stride"), (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
    (dict(x=P + 1), "aligned"), (dict(scale=P + 2), "aligned"), (dict(rows=2**31), "too many"),
])
def test_quantize_refuses(moe, bad, msg):
    _refused(moe, "moe_quantize_int8_async", {**QUANT, **bad}, msg)


INT8MM = dict(x=P, ldx=64, x_dtype=BF16, x_scale=None, w=P, ldw=64, w_stride=64 * 32, w_scale=P, offsets=P, groups=4,
              rows=10, in_dim=64, out_dim=32, y=P, ldy=32, y_dtype=BF16, workspace=P, workspace_bytes=48 + 640, stream=None)


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "groups"), (dict(offsets=None), "offsets"), (dict(x_dtype=FP8), "x_dtype"), (dict(y_dtype=INT8), "result"),
    (dict(in_dim=131072, ldx=131072, ldw=131072), "131071"), (dict(ldx=63), "row stride"), (dict(ldw=63), "row stride"),
    (dict(ldy=31), "row stride"), (dict(w_stride=64 * 31), "w_stride"), (dict(w_scale=None), "null"),
    (dict(x_dtype=INT8), "x_scale"), (dict(workspace=None), "workspace"), (dict(workspace=P + 8), "workspace"),
    (dict(workspace_bytes=48 + 639), "workspace"), (dict(x=P + 1), "aligned"), (dict(w_scale=P + 2), "aligned"),
])
def test_int8_matmul_refuses(moe, bad, msg):
    _refused(moe, "moe_int8_matmul_async", {**INT8MM, **bad}, msg)


NORM = dict(x=P, x_dtype=BF16, y=P, y_dtype=F32, post=P, pre=P, w_dtype=F32, gate=P, gate_dtype=BF16, gate_rows=4,
            alpha=1.0, beta=1.0, eps=1e-5, T=8, D=64, r=P, h=P, h_dtype=BF16, stats=P, stream=None)


@pytest.mark.parametrize("bad,msg", [
    (dict(x_dtype=FP8), "dtypes"), (dict(h_dtype=9), "dtypes"), (dict(T=-1), "T must"), (dict(D=0), "D must"),
    (dict(D=16385), "D must"), (dict(gate_rows=0), "gate_rows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(h=None), "come together"), (dict(pre=None), "come together"), (dict(y=None), "need y"), (dict(x=None), "null"),
    (dict(r=None, h=None, pre=None), "null"), (dict(x=P + 1), "aligned"), (dict(stats=P + 2), "aligned"),
    (dict(T=2**31), "too many"),
])
def test_block_norm_refuses(moe, bad, msg):
    _refused(moe, "moe_block_norm_async", {**NORM, **bad}, msg)


NORMG = dict(dr=P, dh=P, r=P, x_dtype=BF16, y=P, y_dtype=F32, h_dtype=BF16, stats=P, post=P, pre=P, w_dtype=F32, gate=P,
             gate_dtype=BF16, gate_rows=8, alpha=1.0, beta=1.0, T=8, D=64, dx=P, dy=P, dgate=P, dpost=P, dpre=P,
             workspace=P, workspace_bytes=2**30, stream=None)


@pytest.mark.parametrize("bad,msg", [
    (dict(x_dtype=INT8), "dtypes"), (dict(D=16385), "D must"), (dict(y=None), "need y"), (dict(gate=None), "dgate needs"),
    (dict(post=None), "dpost needs"), (dict(pre=None), "dh needs"), (dict(dh=None), "dpre needs"),
    (dict(dr=None, dh=None, dpre=None), "dr or dh"), (dict(r=None), "null"), (dict(stats=None), "null"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace"), (dict(workspace=P + 4), "workspace"),
    (dict(dpost=P + 2), "aligned"), (dict(gate_rows=-1), "gate_rows"),
])
def test_block_norm_grad_refuses(moe, bad, msg):
    _refused(moe, "moe_block_norm_grad_async", {**NORMG, **bad}, msg)


def test_sizes_past_the_32_bit_arithmetic_are_refused(moe):
    from mixtureofexperts_amd import _lib

    big, n = 2**30 + 1, ctypes.c_int64(-1)
    for bad in (dict(rows=big), dict(in_dim=big, ldx=big, ldw=big), dict(out_dim=big, ldy=big, w_stride=64 * big),
                dict(groups=big)):
        _refused(moe, "moe_grouped_matmul_async", {**ROWS, **bad}, "2^30")
    _refused(moe, "moe_grouped_matmul_grad_w_async", {**GRADW, "rows": big}, "2^30")
    _refused(moe, "moe_int8_matmul_async", {**INT8MM, "rows": big}, "2^30")
    _refused(moe, "moe_quantize_int8_async", {**QUANT, "cols": big, "ldx": big, "ldq": big}, "2^30")
    assert _lib.lib().moe_grouped_matmul_workspace(1, big, 8, 8, BF16, ctypes.byref(n)) == _lib.MOE_EINVAL


def test_a_result_on_its_operand_is_refused(moe):
    # square products, so that the sizes alone would allow it
    q = 2 * P
    rows = dict(in_dim=64, out_dim=64, ldy=64, w_stride=64 * 64, dtype=F32, y_dtype=F32)
    for place in (dict(x=P, w=q, y=P), dict(x=P, w=q, y=q)):
        for fn in ("moe_grouped_matmul_async", "moe_grouped_matmul_grad_x_async"):
            _refused(moe, fn, {**ROWS, **rows, **place, "workspace": 4 * P, "workspace_bytes": 2**30}, "overlap")
        args = {**INT8MM, "x": place["x"], "w": place["w"], "y": place["y"], "workspace": 4 * P, "workspace_bytes": 2**30}
        _refused(moe, "moe_int8_matmul_async", args, "overlap")
    for place in (dict(x=P, dy=q, dw=P), dict(x=P, dy=q, dw=q)):
        _refused(moe, "moe_grouped_matmul_grad_w_async", {**GRADW, **place, "workspace": 4 * P, "workspace_bytes": 2**30},
                 "overlap")


def test_empty_calls_are_no_work(moe):
    from mixtureofexperts_amd import _lib

    L = _lib.lib()
    assert L.moe_grouped_matmul_async(*{**ROWS, "rows": 0, "x": None, "y": None}.values()) == 0
    assert L.moe_grouped_matmul_grad_x_async(*{**ROWS, "ldx": 32, "ldy": 64, "rows": 0, "x": None}.values()) == 0
    assert L.moe_quantize_int8_async(*{**QUANT, "rows": 0, "x": None}.values()) == 0
    assert L.moe_int8_matmul_async(*{**INT8MM, "rows": 0, "workspace": None}.values()) == 0
    assert L.moe_block_norm_async(*{**NORM, "T": 0, "x": None}.values()) == 0
    assert L.moe_grouped_matmul_grad_w_async(*{**GRADW, "rows": 0, "accumulate": 1}.values()) == 0


def test_python_refuses_host_tensors(moe):
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 8), torch.zeros(2, 6, 8)
    off = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: moe.grouped_matmul(x, w, off), lambda: moe.grouped_matmul_grad_x(x[:, :6], w, off),
                 lambda: moe.grouped_matmul_grad_w(x, x, off), lambda: moe.quantize_int8(x),
                 lambda: moe.int8_matmul(x, w.to(torch.int8), torch.zeros(2, 6), off),
                 lambda: moe.block_norm(x, pre_weight=torch.ones(8)), lambda: moe.block_norm_grad(x, None, x)):
        with pytest.raises(moe.MoeError, match="GPU memory"):
            call()


@pytest.mark.gpu
def test_python_refuses(moe):
    torch = pytest.importorskip("torch")
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")
    x, w, off = z(4, 8), z(2, 6, 8), z(3, t=torch.int32)
    f32, i8, one = torch.float32, torch.int8, torch.ones(8, device="cuda")
    calls = [
        (lambda: moe.grouped_matmul(x.half(), w, off), "must be"),
        (lambda: moe.grouped_matmul(x, w.float(), off), "must be"),
        (lambda: moe.grouped_matmul(x, w), "offsets are needed"),
        (lambda: moe.grouped_matmul(x, w, off.long()), "must be"),
        (lambda: moe.grouped_matmul(x, w, off[:2]), "contiguous int32"),
        (lambda: moe.grouped_matmul(x[:, :7], w, off), "columns"),
        (lambda: moe.grouped_matmul(x.t(), w, off), "contiguous"),
        (lambda: moe.grouped_matmul(z(1, 8).expand(4, 8), w, off), "overlap"),
        (lambda: moe.grouped_matmul(x, z(1, 6, 8).expand(2, 6, 8), off), "overlap"),
        (lambda: moe.grouped_matmul(x, w, off, layout=3), "layout"),
        (lambda: moe.grouped_matmul(x, w, off, out=z(4, 7)), "out must be"),
        (lambda: moe.grouped_matmul(x, w, off, out_dtype=i8), "result must be"),
        (lambda: moe.grouped_matmul(x.float(), w.float(), off, out_dtype=torch.bfloat16), "result must be"),
        (lambda: moe.grouped_matmul(x, w, off.cpu()), "one device"),
        (lambda: moe.grouped_matmul_grad_w(x, z(5, 6), off), "same rows"),
        (lambda: moe.grouped_matmul_grad_w(x, z(4, 6), off, accumulate=True), "needs out"),
        (lambda: moe.grouped_matmul_grad_w(x, z(4, 6), off[:1]), "two row numbers"),
        (lambda: moe.quantize_int8(z(4, 8, t=i8)), "must be"),
        (lambda: moe.int8_matmul(x, z(2, 6, 8, t=i8), z(2, 5, t=f32), off), "w_scale"),
        (lambda: moe.int8_matmul(z(4, 8, t=i8), z(2, 6, 8, t=i8), z(2, 6, t=f32), off), "x_scale"),
        (lambda: moe.int8_matmul(x, z(2, 6, 8, t=i8), z(2, 6, t=f32), off, x_scale=z(4, t=f32)), "x_scale"),
        (lambda: moe.block_norm(x), "nothing to compute"),
        (lambda: moe.block_norm(x, post_weight=one), "need y"),
        (lambda: moe.block_norm(x, x[:3], post_weight=one), "contiguous"),
        (lambda: moe.block_norm(x, x, pre_weight=one, post_weight=one.bfloat16()), "one type"),
        (lambda: moe.block_norm(x, x, gate=z(3, 8)), "do not divide"),
        (lambda: moe.block_norm(x, x, gate=z(2, 7)), "gate must be"),
        (lambda: moe.block_norm(z(2, 16392), pre_weight=z(16392, t=f32)), "16384"),
        (lambda: moe.block_norm_grad(None, None, x), "dr or dh"),
        (lambda: moe.block_norm_grad(x, x, x), "come together"),
        (lambda: moe.block_norm_grad(x, x, x, pre_weight=one), "stats"),
    ]
    for i, (call, msg) in enumerate(calls):
        with pytest.raises(moe.MoeError, match=msg):
            call()
            print("not refused:", i, flush=True)


@pytest.mark.gpu
def test_python_refuses_no_columns_and_results_in_place(moe):
    torch = pytest.importorskip("torch")
    with pytest.raises(moe.MoeError, match="columns"):
        moe.quantize_int8(torch.zeros(3, 2, 0, device="cuda"))
    x, w = torch.zeros(8, 8, device="cuda"), torch.zeros(8, 8, device="cuda")
    for out in (x, w):
        with pytest.raises(moe.MoeError, match="overlap"):
            moe.grouped_matmul(x, w, out=out)


def test_rows_up_to_2_30(moe):
    # the limit is the documented one: sizes are checked before the pointers, so the
    # largest calls get as far as those (null, or one byte off)
    from mixtureofexperts_amd import _lib

    most, n = 2**30, ctypes.c_int64(-1)
    _refused(moe, "moe_block_norm_async", {**NORM, "T": most, "x": None}, "null")
    _refused(moe, "moe_block_norm_async", {**NORM, "T": most + 1, "x": None}, "2^30")
    _refused(moe, "moe_block_norm_grad_async", {**NORMG, "T": most, "dpost": P + 2}, "aligned")
    _refused(moe, "moe_block_norm_grad_async", {**NORMG, "T": most + 1, "dpost": P + 2}, "2^30")
    _refused(moe, "moe_quantize_int8_async", {**QUANT, "rows": most, "x": None}, "null")
    _refused(moe, "moe_quantize_int8_async", {**QUANT, "rows": most + 1, "x": None}, "2^30")
    _refused(moe, "moe_int8_matmul_async", {**INT8MM, "rows": most, "x": P + 1}, "aligned")
    L = _lib.lib()
    assert L.moe_block_norm_grad_workspace(most, 64, 1, ctypes.byref(n)) == 0 and 0 < n.value < 2**32
    assert L.moe_block_norm_grad_workspace(most + 1, 64, 1, ctypes.byref(n)) == _lib.MOE_EINVAL
    assert L.moe_int8_matmul_workspace(8, most, 64, 32, BF16, ctypes.byref(n)) == 0
    assert n.value >= 4 * most + 64 * most  # scales and codes, past 32 bits


def test_a_result_that_reaches_into_an_operand_is_refused(moe):
    # sizes in elements: x 10 rows of 64, w 4 matrices of 32 x 64, y 10 rows of 32
    ws = dict(workspace=64 * P, workspace_bytes=2**30)
    at = dict(x=P, w=4 * P, offsets=16 * P)
    bf16 = 2
    inside = [P + 64 * bf16, P + 9 * 64 * bf16, P - 32 * bf16 * 10 + bf16,      # within x, its last row, its first element
              4 * P + 3 * 64 * 32 * bf16 + 62, 4 * P - bf16 * 320 + bf16,        # w's last matrix, its first element
              16 * P + 16, 16 * P - 2 * 320 + 2]                                 # the offsets
    for y in inside:
        _refused(moe, "moe_grouped_matmul_async", {**ROWS, **at, **ws, "y": y}, "overlap")
        _refused(moe, "moe_int8_matmul_async",
                 {**INT8MM, **at, **ws, "x_dtype": INT8, "x_scale": 20 * P, "w_scale": 24 * P, "ldx": 128, "ldw": 128,
                  "in_dim": 128, "w_stride": 128 * 32, "y": y}, "overlap")
    for y in (20 * P + 4 * 9, 24 * P + 4 * 127, 24 * P - 320 * bf16 + 2):        # the scales
        _refused(moe, "moe_int8_matmul_async",
                 {**INT8MM, **at, **ws, "x_dtype": INT8, "x_scale": 20 * P, "w_scale": 24 * P, "y": y}, "overlap")
    # columns of one buffer of 96: y's last element is x's first, or x's last y's first
    one = dict(ldx=96, ldy=96)
    for x, y in ((P + 31 * bf16, P), (P, P + 63 * bf16), (P, P + 95 * bf16)):  # (the last wraps into the next row)
        _refused(moe, "moe_grouped_matmul_async", {**ROWS, **at, **ws, **one, "x": x, "y": y}, "overlap")
    # rows of different strides: the fourth of y meets the second of x
    _refused(moe, "moe_grouped_matmul_async", {**ROWS, **at, **ws, "ldx": 1000, "ldy": 300, "y": P + 70 * bf16}, "overlap")
    grad = dict(x=P, dy=4 * P, offsets=16 * P)
    for dw in (P + 4, 4 * P + 10 * 32 * bf16 - 4, 16 * P + 16, P - 4 * 64 * 32 * 4 + 4):
        _refused(moe, "moe_grouped_matmul_grad_w_async", {**GRADW, **grad, **ws, "dw": dw}, "overlap")
    quant = dict(x=P, q=4 * P, scale=8 * P)
    for bad in (dict(q=P + 511), dict(q=P - 255), dict(scale=P + 508), dict(scale=4 * P + 252), dict(scale=4 * P - 12)):
        _refused(moe, "moe_quantize_int8_async", {**QUANT, **quant, **bad}, "overlap")


@pytest.mark.gpu
def test_columns_of_one_buffer_are_taken(moe):
    torch = pytest.importorskip("torch")
    g = torch.Generator(device="cuda").manual_seed(3)
    off = torch.tensor([0, 40, 40, 100], dtype=torch.int32, device="cuda")
    w = torch.randn(3, 32, 64, generator=g, device="cuda")
    buf = torch.randn(100, 64 + 32 + 3, generator=g, device="cuda")
    for x, y in ((buf[:, :64], buf[:, 64:96]), (buf[:, 35:], buf[:, 2:34])):
        want = moe.grouped_matmul(x.contiguous(), w, off)
        keep = x.clone()
        assert torch.equal(moe.grouped_matmul(x, w, off, out=y), want) and torch.equal(x, keep)
    # the weights' gradient beside the weights, the rows in every other row of a buffer
    both = torch.randn(3, 32, 128, generator=g, device="cuda")
    x, dy = torch.randn(200, 64, generator=g, device="cuda"), torch.randn(100, 32, generator=g, device="cuda")
    want = moe.grouped_matmul_grad_w(x[::2].contiguous(), dy, off)
    keep = both[:, :, :64].clone()
    assert torch.equal(moe.grouped_matmul_grad_w(x[::2], dy, off, out=both[:, :, 64:]), want)
    assert torch.equal(both[:, :, :64], keep)
    want = moe.grouped_matmul_grad_x(dy, both[:, :, :64], off)
    assert torch.equal(moe.grouped_matmul_grad_x(dy, both[:, :, :64], off, out=x[1::2]), want)
    # rows of different strides that pass each other
    flat = torch.zeros(100 * 200 + 64, device="cuda")
    x = flat.as_strided((50, 64), (400, 1))
    x.copy_(torch.randn(50, 64, generator=g, device="cuda"))
    y = flat.as_strided((50, 32), (200, 1), 64)
    want = moe.grouped_matmul(x.contiguous(), w[0])
    assert torch.equal(moe.grouped_matmul(x, w[0], out=y), want)
    for x, y in ((x, flat.as_strided((50, 32), (200, 1), 63)), (buf[:50, :64], buf[:50, 63:95])):
        with pytest.raises(moe.MoeError, match="overlap"):
            moe.grouped_matmul(x, w[0], out=y)


def test_more_tiles_than_a_launch_are_refused(moe):
    # the documented limit: no more than 8 million workgroups
    far = dict(x=2**44, w=2**45, offsets=2**46, y=2**56)
    many = dict(rows=2**30, out_dim=2**20, ldy=2**20, w_stride=2**26)
    _refused(moe, "moe_grouped_matmul_async", {**ROWS, **far, **many}, "too many tiles")
    _refused(moe, "moe_grouped_matmul_grad_w_async",
             {**GRADW, "x": 2**44, "dy": 2**45, "offsets": 2**46, "dw": 2**56, "groups": 2**24, "rows": 2**24}, "too many tiles")
    _refused(moe, "moe_int8_matmul_async",
             {**INT8MM, **far, **many, "x_dtype": INT8, "x_scale": 2**43, "w_scale": 2**42, "w_stride": 2**26}, "too many tiles")
