"""Operators on torch tensors in GPU memory: the grouped products of expert
FFNs with their gradients, the gated projections with theirs, int8 products,
8-bit floating point products with a scale per block of 128, and the norms, gate
and residual around a block.  No counterpart in the reference (it has neither gradients nor
integer weights, and its caller does the norms, src/llama2/inference.jl:61).

Every function runs on torch's current stream of the tensors' device, allocates
through torch (workspaces included), does not wait for the GPU and can be
captured into a graph.  Tensors of one call are on one device.  A wrong
argument raises MoeError.

Nothing is recorded for autograd: the gradients are calls of their own, for an
autograd.Function or a training loop that makes them itself.  A tensor that
torch would differentiate (requires_grad while gradients are recorded, or a
forward-mode tangent) is refused, so that no graph is cut unseen: call under
torch.no_grad(), inside a Function, or with detached tensors.

Groups: ``offsets`` is an int32 tensor of E + 1 non-decreasing row numbers on
the device; rows [offsets[e], offsets[e + 1]) belong to expert e, and rows
outside every group are not written and have no effect.  ``None``: one expert, all
rows.  Weights are (E, out, in) with ``layout=MOE_LAYOUT_LLAMA_IN_OUT`` (the
default) and (E, in, out) with ``MOE_LAYOUT_FLUX_OUT_IN``; one expert's may be
2-D.  Rows may be strided (contiguous within a row); 16-byte aligned rows are
read faster.  A result that shares an element with an operand is refused; both
may be columns of one buffer.

Sizes and rows go up to 2^30.  A product is one launch of at most 8 million
workgroups, each with 64 x 64 results or more (few rows per group: 16 columns
of one); what needs more is refused.
"""
import ctypes

from . import _lib
from ._lib import MOE_EINVAL, MOE_LAYOUT_FLUX_OUT_IN, MOE_LAYOUT_LLAMA_IN_OUT
from .activations import activation_code, silu

_torch = _forward_ad = _grad_enabled = _written = None
_codes = {}
_floats = []  # the types of float operands


def _t():
    """torch, imported at first use (the host API needs only numpy)."""
    global _torch, _forward_ad, _grad_enabled, _written
    if _torch is None:
        import torch
        import torch.autograd.forward_ad as forward_ad

        _torch, _forward_ad, _grad_enabled = torch, forward_ad, torch.is_grad_enabled
        _written = torch.autograd.graph.increment_version
        _floats.extend((torch.float32, torch.bfloat16))
        _codes.update({torch.float32: _lib.MOE_F32, torch.bfloat16: _lib.MOE_BF16, torch.int8: _lib.MOE_INT8,
                       torch.float8_e4m3fn: _lib.MOE_FP8_E4M3})
    return _torch


def _bad(msg):
    raise _lib.MoeError(MOE_EINVAL, msg)


def _plain(names, *tensors):
    """Refuses what autograd would have to record (see above); names: the
    arguments', as one string."""
    if _torch is None:
        _t()
    if _grad_enabled():
        try:
            for t in tensors:
                if t is not None and t.requires_grad:
                    name = names.split()[[t is u for u in tensors].index(True)]
                    _bad(f"{name} requires a gradient, which this call does not record: use torch.no_grad() or detach it")
        except AttributeError:
            pass  # not a tensor, which is refused for that
    if _forward_ad._current_level >= 0:  # within a forward_ad.dual_level()
        for name, t in zip(names.split(), tensors):
            if isinstance(t, _torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
                _bad(f"{name} carries a tangent, which this call does not propagate")


def _tensor(t, name, dtypes, dims):
    if not isinstance(t, _t().Tensor) or not t.is_cuda:
        _bad(f"{name} must be a tensor in GPU memory")
    if t.dtype not in dtypes:
        _bad(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() not in dims:
        _bad(f"{name} must have {' or '.join(str(d) for d in dims)} dimensions, got {t.dim()}")
    return t


def _row_stride(t, name):
    """Elements between the rows of t's last two dimensions."""
    rows, cols = t.shape[-2:]
    ld, one = t.stride()[-2:]
    if one != 1 and cols > 1:
        _bad(f"{name}: a row's elements must be contiguous")
    if ld < cols:
        if rows > 1:
            _bad(f"{name}: rows must not overlap")
        ld = cols
    return ld


def _rows(t, name, dtypes):
    """A 2-D tensor of rows: (pointer, row stride)."""
    _tensor(t, name, dtypes, (2,))
    if max(t.shape) > 2**31 - 1:
        _bad(f"{name}: sizes must fit 32 bits")
    return t.data_ptr(), _row_stride(t, name)


def _matrices(t, name, dtypes=None):
    """(E, a, b) or (a, b): (E, a, b, row stride, matrix stride); without dtypes
    of a tensor that is checked already."""
    if dtypes is not None:
        _tensor(t, name, dtypes, (2, 3))
        if max(t.shape) > 2**31 - 1:
            _bad(f"{name}: sizes must fit 32 bits")
    a, b = t.shape[-2:]
    ld = _row_stride(t, name)
    if t.dim() == 2:
        return 1, a, b, ld, 0
    E = t.shape[0]
    stride = t.stride(0) if E > 1 else 0
    if E > 1 and stride < (a - 1) * ld + b:
        _bad(f"{name}: matrices must not overlap")
    return E, a, b, ld, stride


def _offsets(offsets, E):
    if offsets is None:
        if E != 1:
            _bad("offsets are needed for more than one expert")
        return None
    torch = _t()
    _tensor(offsets, "offsets", (torch.int32,), (1,))
    if offsets.shape[0] != E + 1 or not offsets.is_contiguous():
        _bad(f"offsets must be {E + 1} contiguous int32")
    return offsets.data_ptr()


def _same_device(first, *tensors):
    """The device of all tensors (None: left out), `first` among them."""
    device = first.device
    for t in tensors:
        if t is not None and t.device != device:
            _bad("tensors must be on one device")
    return device


def _call(fn, device, *args):
    """The library call on `device`'s current stream (its last argument)."""
    # torch's own binding: building a torch.cuda.Stream costs 3 us, as much as the launch
    index, cuda = device.index, _torch._C
    if index != cuda._cuda_getDevice():
        with _torch.cuda.device(device):
            return _call(fn, device, *args)
    status = fn(*args, cuda._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status)


_workspace_bytes = {}  # (query, device, sizes) -> bytes: a function of the sizes and the GPU's CUs


def _workspace(fn, device, *sizes):
    """(tensor or None, its address, its bytes) as the library's query asks."""
    key = (fn.__name__, device.index, sizes)
    n = _workspace_bytes.get(key)
    if n is None:
        need = ctypes.c_int64(0)
        with _torch.cuda.device(device):
            _lib.check(fn(*sizes, ctypes.byref(need)))
        if len(_workspace_bytes) >= 4096:
            _workspace_bytes.clear()
        n = _workspace_bytes[key] = need.value
    if n == 0:
        return None, None, 0
    ws = _torch.empty(n, dtype=_torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def _layout(layout):
    if layout not in (MOE_LAYOUT_LLAMA_IN_OUT, MOE_LAYOUT_FLUX_OUT_IN):
        _bad("unknown layout")
    return layout == MOE_LAYOUT_FLUX_OUT_IN


def _result(out, shape, dtype, dtypes, like, clear):
    """The caller's `out`, checked, or a new tensor (zeros where a call may
    leave elements unwritten)."""
    torch = _torch
    if out is None:
        if dtype not in dtypes:
            _bad(f"the result must be {' or '.join(str(d) for d in dtypes)}, got {dtype}")
        return (torch.zeros if clear else torch.empty)(shape, dtype=dtype, device=like.device)
    _tensor(out, "out", dtypes, (len(shape),))
    if out.shape != shape:
        _bad(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    if dtype is not None and out.dtype != dtype:
        _bad("out and out_dtype differ")
    return out


def _float_types(dtype):
    """The results that operands of dtype may have."""
    return (dtype,) if dtype == _torch.float32 else _floats


def _rows_product(fn, x, name, names, w, offsets, layout, out, out_dtype, grad):
    _plain(names, x, w, out)
    xp, ldx = _rows(x, name, _floats)
    E, a, b, ldw, stride = _matrices(w, "w", (x.dtype,))
    in_dim, out_dim = (a, b) if _layout(layout) else (b, a)
    k, n = (out_dim, in_dim) if grad else (in_dim, out_dim)
    if x.shape[1] != k:
        _bad(f"{name} has {x.shape[1]} columns, the weights take {k}")
    if out is None and out_dtype is None:
        out_dtype = x.dtype
    given = out
    out = _result(out, (x.shape[0], n), out_dtype, _float_types(x.dtype), x, offsets is not None)
    device, M, dt = _same_device(x, w, offsets, out), x.shape[0], _codes[x.dtype]
    ws, wsp, wsn = _workspace(_lib.lib().moe_grouped_matmul_workspace, device, E, M, in_dim, out_dim, dt)
    _call(fn, device, xp, ldx, w.data_ptr(), ldw, stride, layout, _offsets(offsets, E), E, M, in_dim, out_dim, dt,
          out.data_ptr(), _row_stride(out, "out"), _codes[out.dtype], wsp, wsn)
    if given is not None:
        _written(out)  # autograd sees the caller's tensor change
    return out


def grouped_matmul(x, w, offsets=None, *, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None, out_dtype=None):
    """y[r] = W_e x[r] for the rows r of expert e: x (M, in) float32 or
    bfloat16, w of the same type; sums in float32, the result in x's type or,
    for bfloat16, ``out_dtype=torch.float32``.  Without ``out`` rows outside
    every group are zeros."""
    return _rows_product(_lib.lib().moe_grouped_matmul_async, x, "x", "x w out", w, offsets, layout, out, out_dtype,
                         False)


def grouped_matmul_grad_x(dy, w, offsets=None, *, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None, out_dtype=None):
    """The gradient of grouped_matmul with respect to x: dx[r] = W_e' dy[r]."""
    return _rows_product(_lib.lib().moe_grouped_matmul_grad_x_async, dy, "dy", "dy w out", w, offsets, layout, out,
                         out_dtype, True)


def grouped_matmul_grad_w(x, dy, offsets=None, *, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None, out_dtype=None,
                          accumulate=False):
    """The gradient of grouped_matmul with respect to w, in ``layout``: for each
    expert the sum over its rows of dy[r] x[r]'; zeros for an expert without
    rows.  ``accumulate`` adds to what ``out`` holds (in float32, rounded
    once)."""
    torch = _t()
    _plain("x dy out", x, dy, out)
    L = _lib.lib()
    xp, ldx = _rows(x, "x", _floats)
    dp, lddy = _rows(dy, "dy", (x.dtype,))
    if x.shape[0] != dy.shape[0]:
        _bad("x and dy must have the same rows")
    if accumulate and out is None:
        _bad("accumulate needs out")
    E = 1 if offsets is None else _tensor(offsets, "offsets", (torch.int32,), (1,)).shape[0] - 1
    if E < 1:
        _bad("offsets must hold at least two row numbers")
    a, b = (x.shape[1], dy.shape[1]) if _layout(layout) else (dy.shape[1], x.shape[1])
    if out is None and out_dtype is None:
        out_dtype = x.dtype
    shape = (a, b) if (out.dim() == 2 if out is not None else offsets is None) and E == 1 else (E, a, b)
    given = out
    out = _result(out, shape, out_dtype, _float_types(x.dtype), x, False)
    _, _, _, ldw, stride = _matrices(out, "out")
    device = _same_device(x, dy, offsets, out)
    ws, wsp, wsn = _workspace(L.moe_grouped_matmul_grad_w_workspace, device, E, x.shape[0], x.shape[1], dy.shape[1])
    _call(L.moe_grouped_matmul_grad_w_async, device, xp, ldx, dp, lddy, layout, _offsets(offsets, E), E, x.shape[0],
          x.shape[1], dy.shape[1], _codes[x.dtype], out.data_ptr(), ldw, stride, _codes[out.dtype], int(accumulate),
          wsp, wsn)
    if given is not None:
        _written(out)  # autograd sees the caller's tensor change
    return out


def _results(out, names, shape, dtypes, allowed, like, clear):
    """The caller's tensors `out` (None: new ones) for the results `names`, checked."""
    if out is None:
        return tuple(_result(None, shape, t, a, like, clear) for t, a in zip(dtypes, allowed))
    if not isinstance(out, (tuple, list)) or len(out) != len(names):
        _bad(f"out must be ({', '.join(names)})")
    for t, name, dtype, a in zip(out, names, dtypes, allowed):
        _tensor(t, name, a, (2,))
        if t.shape != shape:
            _bad(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
        if dtype is not None and t.dtype != dtype:
            _bad("out and out_dtype differ")
    return tuple(out)


def _two_weights(w1, w3, dtype):
    """w1 and w3 of one shape: (E, a, b), (pointer, row stride, matrix stride) of each."""
    E, a, b, ld1, s1 = _matrices(w1, "w1", (dtype,))
    ld3, s3 = ld1, s1
    _tensor(w3, "w3", (dtype,), (2, 3))
    if w3.shape != w1.shape or w3.stride() != w1.stride():
        E3, a3, b3, ld3, s3 = _matrices(w3, "w3")
        if (E3, a3, b3) != (E, a, b):
            _bad(f"w1 and w3 must have one shape, got {tuple(w1.shape)} and {tuple(w3.shape)}")
    return E, a, b, (w1.data_ptr(), ld1, s1, w3.data_ptr(), ld3, s3)


def gated_matmul(x, w1, w3, offsets=None, *, activation=silu, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None, out_dtype=None,
                 save=False):
    """The two projections of a gated feed-forward block, its activation and the
    product in one kernel: h[r] = act(a[r]) * b[r], a[r] = W1_e x[r], b[r] = W3_e x[r]
    for the rows r of expert e.  x (M, in) float32 or bfloat16, w1 and w3 of the
    same type; activation silu, gelu (tanh form), relu or identity; sums and gate in
    float32; h in x's type or, for bfloat16, ``out_dtype=torch.float32``.  With
    ``save`` (h, a, b), a and b in x's type, as gated_matmul_grad takes them; ``out``
    is then a tuple of the three.  Without ``out`` rows outside every group are
    zeros."""
    given = out
    _plain("x w1 w3 out out out", x, w1, w3, *(out if isinstance(out, (tuple, list)) else (out,)))
    act = activation_code(activation)
    xp, ldx = _rows(x, "x", _floats)
    E, a, b, w = _two_weights(w1, w3, x.dtype)
    k, n = (a, b) if _layout(layout) else (b, a)
    if x.shape[1] != k:
        _bad(f"x has {x.shape[1]} columns, the weights take {k}")
    M, dt, shape = x.shape[0], _codes[x.dtype], (x.shape[0], n)
    if out is None and out_dtype is None:
        out_dtype = x.dtype
    pa = pb = None
    lda = ldb = 0
    if save:
        kept = (x.dtype,)
        res = _results(out, ("h", "a", "b"), shape, (out_dtype, x.dtype, x.dtype), (_float_types(x.dtype), kept, kept), x,
                       offsets is not None)
        h, ta, tb = res
        device = _same_device(x, w1, w3, offsets, h, ta, tb)
        pa, lda, pb, ldb = ta.data_ptr(), _row_stride(ta, "a"), tb.data_ptr(), _row_stride(tb, "b")
    else:
        h = _result(out, shape, out_dtype, _float_types(x.dtype), x, offsets is not None)
        res = (h,)
        device = _same_device(x, w1, w3, offsets, h)
    L = _lib.lib()
    ws, wsp, wsn = _workspace(L.moe_gated_matmul_workspace, device, E, M, k, n, dt)
    _call(L.moe_gated_matmul_async, device, xp, ldx, *w, layout, act, _offsets(offsets, E), E, M, k, n, dt,
          h.data_ptr(), _row_stride(h, "out"), _codes[h.dtype], pa, lda, pb, ldb, wsp, wsn)
    if given is not None:
        for t in res:
            _written(t)  # autograd sees the caller's tensors change
    return res if save else h


def gated_matmul_grad(dy, a, b, w2=None, offsets=None, *, activation=silu, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None):
    """The gradients of a gated block y[r] = W2_e h[r], h = act(a) * b with respect to
    a and b, from dy (M, out) and what gated_matmul saved:

        dh = W2' dy,  da = dh * b * act'(a),  db = dh * act(a)

    Returns (da, db, h), all in dy's type: h is formed again for the gradient of W2.
    dh stays in float32 and is not stored.  w2 (E, out, hidden) in ``layout``; without
    it dy is dh itself (M, hidden).  The rest of the backward pass: dx is
    gated_matmul_grad_x(da, db, w1, w3, ...), the gradients of w1, w3 and w2 are
    grouped_matmul_grad_w of (x, da), (x, db) and (h, dy).  ``out`` is a tuple (da, db,
    h); without it rows outside every group are zeros."""
    given = out
    _plain("dy a b w2 out out out", dy, a, b, w2, *(out if isinstance(out, (tuple, list)) else (out,)))
    act = activation_code(activation)
    dp, lddy = _rows(dy, "dy", _floats)
    kept = (dy.dtype,)
    ap, lda = _rows(a, "a", kept)
    bp, ldb = _rows(b, "b", kept)
    M, n = a.shape
    if b.shape != a.shape or dy.shape[0] != M:
        _bad("a and b must have one shape, and dy their rows")
    if w2 is None:
        _layout(layout)
        E = 1 if offsets is None else _tensor(offsets, "offsets", (_torch.int32,), (1,)).shape[0] - 1
        if E < 1:
            _bad("offsets must hold at least two row numbers")
        k, w = n, (None, 0, 0)
    else:
        E, p, q, ldw, stride = _matrices(w2, "w2", kept)
        hidden, k = (p, q) if _layout(layout) else (q, p)
        if hidden != n:
            _bad(f"a has {n} columns, w2 takes {hidden}")
        w = (w2.data_ptr(), ldw, stride)
    if dy.shape[1] != k:
        _bad(f"dy has {dy.shape[1]} columns, " + (f"w2 gives {k}" if w2 is not None else f"without w2 it is dh, of {n}"))
    dt = _codes[dy.dtype]
    res = _results(out, ("da", "db", "h"), a.shape, (dy.dtype,) * 3, (kept,) * 3, a, offsets is not None)
    device = _same_device(dy, a, b, w2, offsets, *res)
    ws, wsp, wsn = None, None, 0
    if w2 is not None:
        ws, wsp, wsn = _workspace(_lib.lib().moe_gated_matmul_grad_workspace, device, E, M, n, k, dt)
    to = [v for t, name in zip(res, ("da", "db", "h")) for v in (t.data_ptr(), _row_stride(t, name))]
    _call(_lib.lib().moe_gated_matmul_grad_async, device, dp, lddy, *w, layout, act, ap, lda, bp, ldb, _offsets(offsets, E),
          E, M, n, k, dt, *to, wsp, wsn)
    if given is not None:
        for t in res:
            _written(t)  # autograd sees the caller's tensors change
    return res


def gated_matmul_grad_x(da, db, w1, w3, offsets=None, *, layout=MOE_LAYOUT_LLAMA_IN_OUT, out=None, out_dtype=None):
    """The gradient of gated_matmul with respect to x, both projections in one sum:
    dx[r] = W1_e' da[r] + W3_e' db[r]; da and db (M, hidden) of the weights' type, the
    result as grouped_matmul's."""
    _plain("da db w1 w3 out", da, db, w1, w3, out)
    ap, lda = _rows(da, "da", _floats)
    bp, ldb = _rows(db, "db", (da.dtype,))
    if db.shape != da.shape:
        _bad("da and db must have one shape")
    E, a, b, w = _two_weights(w1, w3, da.dtype)
    k, n = (a, b) if _layout(layout) else (b, a)
    if da.shape[1] != n:
        _bad(f"da has {da.shape[1]} columns, the weights give {n}")
    M, dt = da.shape[0], _codes[da.dtype]
    if out is None and out_dtype is None:
        out_dtype = da.dtype
    given = out
    out = _result(out, (M, k), out_dtype, _float_types(da.dtype), da, offsets is not None)
    device = _same_device(da, db, w1, w3, offsets, out)
    ws, wsp, wsn = _workspace(_lib.lib().moe_gated_matmul_grad_x_workspace, device, E, M, k, n, dt)
    _call(_lib.lib().moe_gated_matmul_grad_x_async, device, ap, lda, bp, ldb, *w, layout, _offsets(offsets, E), E, M, k, n, dt,
          out.data_ptr(), _row_stride(out, "out"), _codes[out.dtype], wsp, wsn)
    if given is not None:
        _written(out)  # autograd sees the caller's tensor change
    return out


def quantize_int8(x):
    """int8 codes with a scale per row: x (..., cols) float32 or bfloat16 ->
    (codes int8 of x's shape, scales float32 (...)).  scale = max|row| / 127,
    code = 127 x / max|row| rounded to nearest even; a row of zeros has scale 0,
    one that holds an infinity or a NaN scale NaN.  Of a weight (E, out, in)
    this gives the codes and scales that int8_matmul takes."""
    torch = _t()
    _plain("x", x)
    _tensor(x, "x", _floats, range(1, 9))
    if not 1 <= x.shape[-1] < 2**31:
        _bad("x must have 1 to 2^31 - 1 columns")
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call(_lib.lib().moe_quantize_int8_async, x.device, x2.data_ptr(), _row_stride(x2, "x"), _codes[x.dtype],
          x2.shape[0], x2.shape[1], q.data_ptr(), x2.shape[1], scale.data_ptr())
    return q, scale


def int8_matmul(x, w, w_scale, offsets=None, *, x_scale=None, out=None, out_dtype=None):
    """y[r][n] = x_scale[r] w_scale[e][n] sum_k q[r][k] w[e][n][k], the sum exact
    in int32.  x (M, in): int8 codes with ``x_scale`` (M,), or float32 /
    bfloat16 rows, which are quantised as quantize_int8 does; w (E, out, in) int8
    and w_scale (E, out) float32 from quantize_int8.  The result is bfloat16 or,
    with ``out_dtype``, float32; without ``out`` rows outside every group are
    zeros."""
    torch = _t()
    _plain("x w_scale x_scale out", x, w_scale, x_scale, out)
    L = _lib.lib()
    xp, ldx = _rows(x, "x", (torch.float32, torch.bfloat16, torch.int8))
    E, n, k, ldw, stride = _matrices(w, "w", (torch.int8,))
    if x.shape[1] != k:
        _bad(f"x has {x.shape[1]} columns, the weights take {k}")
    _tensor(w_scale, "w_scale", (torch.float32,), (w.dim() - 1,))
    if w_scale.shape != w.shape[:-1] or not w_scale.is_contiguous():
        _bad(f"w_scale must be contiguous {tuple(w.shape[:-1])}")
    codes = x.dtype == torch.int8
    if codes != (x_scale is not None):
        _bad("x_scale belongs to int8 rows")
    if codes:
        _tensor(x_scale, "x_scale", (torch.float32,), (1,))
        if x_scale.shape[0] != x.shape[0] or not x_scale.is_contiguous():
            _bad("x_scale must be contiguous with one scale per row")
    if out is None and out_dtype is None:
        out_dtype = torch.bfloat16
    given = out
    out = _result(out, (x.shape[0], n), out_dtype, (torch.bfloat16, torch.float32), x, offsets is not None)
    device = _same_device(x, w, w_scale, x_scale, offsets, out)
    ws, wsp, wsn = _workspace(L.moe_int8_matmul_workspace, device, E, x.shape[0], k, n, _codes[x.dtype])
    _call(L.moe_int8_matmul_async, device, xp, ldx, _codes[x.dtype], x_scale.data_ptr() if codes else None,
          w.data_ptr(), ldw, stride, w_scale.data_ptr(), _offsets(offsets, E), E, x.shape[0], k, n, out.data_ptr(),
          _row_stride(out, "out"), _codes[out.dtype], wsp, wsn)
    if given is not None:
        _written(out)  # autograd sees the caller's tensor change
    return out


def quantize_fp8(x, *, block_rows=1):
    """8-bit floating point codes (torch.float8_e4m3fn) with a float32 scale for each
    block of 128: x (..., cols) float32 or bfloat16 -> (codes of x's shape, scales).
    block_rows=1: a scale for each 128 elements of a row, (..., ceil(cols / 128)), as
    fp8_matmul takes rows.  block_rows=128: x (E, rows, cols) or (rows, cols), a scale
    for each 128 x 128 block, (E, ceil(rows / 128), ceil(cols / 128)), as it takes weights.
    scale = max|block| / 448, code = 448 x / max|block| rounded to nearest even, exactly; a
    block of zeros has scale 0, one that holds an infinity or a NaN scale NaN."""
    torch = _t()
    _plain("x", x)
    if block_rows not in (1, 128):
        _bad("block_rows must be 1 or 128")
    _tensor(x, "x", _floats, range(1, 9) if block_rows == 1 else (2, 3))
    cols = x.shape[-1]
    if not 1 <= cols < 2**31:
        _bad("x must have 1 to 2^31 - 1 columns")
    kb = -(-cols // 128)
    if block_rows == 1:
        x2 = x.reshape(-1, cols) if x.dim() != 2 else x
        E, rows, ldx, stride = 1, x2.shape[0], _row_stride(x2, "x"), 0
        shape = (*x.shape[:-1], kb)
    else:
        x2 = x
        E, rows, _, ldx, stride = _matrices(x, "x")
        shape = (*x.shape[:-2], -(-rows // 128), kb)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(shape, dtype=torch.float32, device=x.device)
    _call(_lib.lib().moe_quantize_fp8_async, x.device, x2.data_ptr(), ldx, stride, _codes[x.dtype], E, rows, cols, block_rows,
          q.data_ptr(), cols, rows * cols, scale.data_ptr())
    return q, scale


def fp8_matmul(x, w, w_scale, offsets=None, *, x_scale=None, out=None, out_dtype=None, exact=False):
    """y[r][n] = sum_k (q[r][k] x_scale[r][k / 128]) (w[e][n][k] w_scale[e][n / 128][k / 128])
    for the rows r of expert e.  x (M, in): float8_e4m3fn codes with ``x_scale`` (M,
    ceil(in / 128)), or float32 / bfloat16 rows, which are quantised as quantize_fp8 does;
    w (E, out, in) float8_e4m3fn and w_scale from quantize_fp8(w, block_rows=128).  A
    block's products are summed in float32, scaled, and summed in float32.  The result is
    bfloat16 or, with ``out_dtype``, float32.  On the way to a bfloat16 result of more than a
    few rows the matrix unit's 8-bit instruction cuts a product to a multiple of 2^-13 of the
    largest of eight (a sum of N(0, 1) codes is off by 1.4e-5 of itself, any sum by less than
    7 * 2^-13 of its magnitudes); with ``exact`` the products are exact whatever the rows, and
    a bfloat16 result is the float32 one rounded, at half the matrix rate.  Without ``out``
    rows outside every group are zeros.  The gradient with respect to x is the same call on
    dy with the transposed codes and scales (w.transpose(1, 2).contiguous()): a matrix' 128 x
    128 blocks are those of its transpose."""
    torch = _t()
    _plain("x w w_scale x_scale out", x, w, w_scale, x_scale, out)
    L, f8 = _lib.lib(), torch.float8_e4m3fn
    xp, ldx = _rows(x, "x", (torch.float32, torch.bfloat16, f8))
    E, n, k, ldw, stride = _matrices(w, "w", (f8,))
    if x.shape[1] != k:
        _bad(f"x has {x.shape[1]} columns, the weights take {k}")
    M, kb = x.shape[0], -(-k // 128)
    _tensor(w_scale, "w_scale", (torch.float32,), (w.dim(),))
    if w_scale.shape != (*w.shape[:-2], -(-n // 128), kb) or not w_scale.is_contiguous():
        _bad(f"w_scale must be contiguous {(*w.shape[:-2], -(-n // 128), kb)}")
    codes = x.dtype == f8
    if codes != (x_scale is not None):
        _bad("x_scale belongs to float8 rows")
    if codes:
        _tensor(x_scale, "x_scale", (torch.float32,), (2,))
        if x_scale.shape != (M, kb) or not x_scale.is_contiguous():
            _bad(f"x_scale must be contiguous {(M, kb)}")
    if out is None and out_dtype is None:
        out_dtype = torch.bfloat16
    given = out
    out = _result(out, (M, n), out_dtype, (torch.bfloat16, torch.float32), x, offsets is not None)
    device = _same_device(x, w, w_scale, x_scale, offsets, out)
    ws, wsp, wsn = _workspace(L.moe_fp8_matmul_workspace, device, E, M, k, n, _codes[x.dtype])
    fn = L.moe_fp8_matmul_exact_async if exact else L.moe_fp8_matmul_async
    _call(fn, device, xp, ldx, _codes[x.dtype], x_scale.data_ptr() if codes else None, w.data_ptr(), ldw, stride,
          w_scale.data_ptr(), _offsets(offsets, E), E, M, k, n, out.data_ptr(), _row_stride(out, "out"), _codes[out.dtype],
          wsp, wsn)
    if given is not None:
        _written(out)  # autograd sees the caller's tensor change
    return out


def _dense(t, name, dtypes, shape):
    """The address of a contiguous tensor of the given shape (None of None)."""
    if t is None:
        return None
    if not (isinstance(t, _torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.shape == shape and t.is_contiguous()):
        _tensor(t, name, dtypes, range(1, 9))
        _bad(f"{name} must be contiguous {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _norm_params(D, T, pre_weight, post_weight, gate):
    """Checks shared by block_norm and its gradient: the weights' addresses and
    type code, the gate's address, type code and rows per gate row."""
    shape = (D,)
    pre, post = _dense(pre_weight, "pre_weight", _floats, shape), _dense(post_weight, "post_weight", _floats, shape)
    wt = _lib.MOE_F32
    if pre_weight is not None or post_weight is not None:
        wt = _codes[(pre_weight if pre_weight is not None else post_weight).dtype]
        if pre_weight is not None and post_weight is not None and pre_weight.dtype != post_weight.dtype:
            _bad("pre_weight and post_weight must have one type")
    if gate is None:
        return pre, post, wt, None, 0, 0
    _tensor(gate, "gate", _floats, (1, 2))
    gates = gate.shape[0] if gate.dim() == 2 else 1
    if gate.shape[-1] != D or not gate.is_contiguous():
        _bad(f"gate must be contiguous (gates, {D}) or ({D},)")
    if gates < 1 or T % gates:
        _bad(f"{T} rows do not divide among {gates} gate rows")
    return pre, post, wt, gate.data_ptr(), _codes[gate.dtype], max(1, T // gates)


def _ptr(t):
    return None if t is None else t.data_ptr()


def block_norm(x, y=None, *, pre_weight=None, post_weight=None, gate=None, alpha=1.0, beta=1.0, eps=1e-5,
               h_dtype=None):
    """The norms before and after a block with its gate and the residual:

        z = y * rstd(y) * post_weight     (without post_weight: y)
        r = alpha x + beta gate * z       (without gate: 1; without y: alpha x)
        h = r * rstd(r) * pre_weight      (without pre_weight: no h)

    over the last dimension D (at most 16384), rstd(v) = 1 / sqrt(mean(v^2) +
    eps).  x (..., D) is the residual stream, y the block's output, r the stream
    after it and h what the next block reads, in ``h_dtype`` (x's type if not
    given); float32 or bfloat16 each.  gate (D,), or (G, D) with each of its
    rows for the next T / G of the T rows.  Returns (r, h, stats); stats (T, 2)
    is what block_norm_grad needs.  Without y and with alpha 1 r is x."""
    torch = _t()
    _plain("x y pre_weight post_weight gate", x, y, pre_weight, post_weight, gate)
    _tensor(x, "x", _floats, range(1, 9))
    shape = x.shape
    D = shape[-1]
    if D < 1:
        _bad("x has no channels")
    T = x.numel() // D
    if not x.is_contiguous():
        _bad(f"x must be contiguous {tuple(shape)}")
    xp, yp = x.data_ptr(), _dense(y, "y", _floats, shape)
    if y is None:
        if post_weight is not None or gate is not None:
            _bad("post_weight and gate need y")
        if pre_weight is None:
            _bad("nothing to compute: give y or pre_weight")
    pre, post, wt, gp, gt, gate_rows = _norm_params(D, T, pre_weight, post_weight, gate)
    xt = x.dtype
    h_dtype = xt if h_dtype is None else h_dtype
    if h_dtype not in _floats:
        _bad("h_dtype must be float32 or bfloat16")
    device = _same_device(x, y, pre_weight, post_weight, gate)
    r = x if y is None and alpha == 1.0 else torch.empty_like(x)
    h = None
    if pre is not None:
        h = torch.empty_like(x) if h_dtype == xt else torch.empty(shape, dtype=h_dtype, device=device)
    stats = torch.empty((T, 2), dtype=torch.float32, device=device)
    _call(_lib.lib().moe_block_norm_async, device, xp, _codes[xt], yp, _codes[y.dtype] if y is not None else 0, post, pre,
          wt, gp, gt, gate_rows, alpha, beta, eps, T, D, None if r is x else r.data_ptr(), _ptr(h), _codes[h_dtype],
          stats.data_ptr())
    return r, h, stats


def block_norm_grad(dr, dh, r, y=None, stats=None, *, pre_weight=None, post_weight=None, gate=None, alpha=1.0,
                    beta=1.0):
    """Gradients of block_norm from dr and dh (None: 0), with its r and stats:
    (dx, dy, dgate, dpost, dpre), None for what the call does not have; dx in
    r's type, dy in y's, the others float32."""
    torch = _t()
    _plain("dr dh r y stats pre_weight post_weight gate", dr, dh, r, y, stats, pre_weight, post_weight, gate)
    L = _lib.lib()
    _tensor(r, "r", _floats, range(1, 9))
    shape = r.shape
    D = shape[-1]
    if D < 1:
        _bad("r has no channels")
    T = r.numel() // D
    if not r.is_contiguous():
        _bad(f"r must be contiguous {tuple(shape)}")
    rp, drp = r.data_ptr(), _dense(dr, "dr", (r.dtype,), shape)
    dhp, yp = _dense(dh, "dh", _floats, shape), _dense(y, "y", _floats, shape)
    sp = _dense(stats, "stats", (torch.float32,), (T, 2))
    if dr is None and dh is None:
        _bad("dr or dh is needed")
    if (dh is not None) != (pre_weight is not None):
        _bad("dh and pre_weight come together")
    if y is None and (post_weight is not None or gate is not None):
        _bad("post_weight and gate need y")
    if stats is None and (pre_weight is not None or post_weight is not None):
        _bad("stats are needed")
    pre, post, wt, gp, gt, gate_rows = _norm_params(D, T, pre_weight, post_weight, gate)
    device = _same_device(r, dr, dh, y, stats, pre_weight, post_weight, gate)
    dx = torch.empty_like(r)
    dy = torch.empty_like(y) if y is not None else None
    # (a sum over no rows is zero; the call writes a gate row's sum with its rows)
    new = lambda size: (torch.empty if T else torch.zeros)(size, dtype=torch.float32, device=device)
    dgate = new(gate.shape) if gate is not None else None
    dpost = new(D) if post is not None else None
    dpre = new(D) if pre is not None else None
    ws, wsp, wsn = None, None, 0
    if dgate is not None or dpost is not None or dpre is not None:
        ws, wsp, wsn = _workspace(L.moe_block_norm_grad_workspace, device, T, D, gate_rows)
    _call(L.moe_block_norm_grad_async, device, drp, dhp, rp, _codes[r.dtype], yp, _codes[y.dtype] if y is not None else 0,
          _codes[dh.dtype] if dh is not None else 0, sp, post, pre, wt, gp, gt, gate_rows, alpha, beta, T, D,
          dx.data_ptr(), _ptr(dy), _ptr(dgate), _ptr(dpost), _ptr(dpre), wsp, wsn)
    return dx, dy, dgate, dpost, dpre
