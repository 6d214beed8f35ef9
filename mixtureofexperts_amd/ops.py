"""Operators on torch tensors in GPU memory: the grouped products of expert
FFNs with their gradients, int8 products, and the norms, gate and residual
around a block.  No counterpart in the reference (it has neither gradients nor
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
        _codes.update({torch.float32: _lib.MOE_F32, torch.bfloat16: _lib.MOE_BF16, torch.int8: _lib.MOE_INT8})
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
