"""The operators beside the MoE layer that work on a caller's own device
tensors, and the calls by which their speed is judged:

  op "fwd"        y[r] = W_e x[r] for the rows r of group e (rows sorted by expert)
  op "grad_x"     dx[r] = W_e^T dy[r]
  op "grad_w"     dW_e = sum over the rows of group e of dy[r] x[r]^T
  op "int8"       x quantised per row, times int8 matrices with a scale per output channel
  op "norm"       r = alpha x + beta gate norm(y) w_post, h = norm(r) w_pre
  op "norm_grad"  the gradients of "norm" with respect to x, y, the gate and both weights

M rows in E groups (`skew`: how uneven the groups are; `tail`: rows behind the
last group, which stay as they were), each row of K inputs and N outputs; `w`
the operands' type, `o` the result's; `layout` the weight's memory order
("llama": [out][in], "flux": [in][out]); `pad` elements between rows.  The
norms take M rows of N channels; `x`, `y`, `h` the types of the residual
stream, of the block's output and of the normed rows; `gate` the rows that
share a gate row (0: no gate); `pre` / `post` which of the norms are there.
"""
import math

import numpy as np
import torch

own = False

_MM = dict(op="fwd", M=1, E=1, K=64, N=64, w="bf16", o="bf16", layout="llama", skew="none", tail=0, pad=0)
_NORM = dict(op="norm", M=1, N=512, x="bf16", y="f32", h="bf16", gate=0, pre=True, post=True)
_ALPHA, _BETA, _EPS = 0.875, 1.25, 1e-5


def _case(name, **kw):
    c = dict(_NORM if kw["op"].startswith("norm") else _MM, **kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # the README layer's up product (32 tokens, top-2 of 8 experts, 512 -> 2048)
        # at reference precision: few rows per expert, every expert's matrix read
        _case("fwd_readme_f32", op="fwd", M=64, E=8, K=512, N=2048, w="f32", o="f32", skew="normal"),
        # a decode step of sixteen sequences on a Mixtral-8x7B-sized layer: four rows
        # per expert, bound by reading the weights
        _case("fwd_mixtral_decode", op="fwd", M=32, E=8, K=4096, N=14336, skew="normal"),
        # the same layer's up product over a full training batch
        _case("fwd_mixtral", op="fwd", M=8192, E=8, K=4096, N=14336, skew="normal"),
        # its down product's input gradient: the weight read along its other side
        _case("grad_x_mixtral", op="grad_x", M=8192, E=8, K=14336, N=4096, skew="normal"),
        # fine-grained experts in training: the weight gradient over ragged groups
        # under a Zipf load, summed into an fp32 result, rows padded behind the last group
        _case("grad_w_deepseek", op="grad_w", M=49152, E=64, K=2048, N=1408, o="f32", skew="zipf", tail=512),
        # odd sizes everywhere at reference precision: the weight gradient of the
        # up product, no dimension a multiple of a tile
        _case("grad_w_ragged_f32", op="grad_w", M=3111, E=12, K=1001, N=2731, w="f32", o="f32", layout="flux",
              skew="zipf"),
        # one token of that Mixtral layer served with int8 weights: two rows, two experts
        _case("int8_mixtral_token", op="int8", M=2, E=8, K=4096, N=14336),
        # a prompt on the int8 experts
        _case("int8_mixtral", op="int8", M=8192, E=8, K=4096, N=14336, skew="normal"),
        # a short ragged prompt on fine-grained int8 experts
        _case("int8_deepseek_517", op="int8", M=3102, E=64, K=1408, N=2048, o="f32", skew="zipf"),
        # one token between two blocks of a stories42M-sized Llama2: latency
        _case("norm_stories42m", op="norm", M=1, N=512, x="f32", y="f32", h="f32", post=False),
        # a training batch between two Mixtral-sized blocks, a gate per channel; y is
        # the MoE layer's fp32 output
        _case("norm_mixtral", op="norm", M=8192, N=4096, gate=8192),
        # the gradients of the same
        _case("norm_grad_mixtral", op="norm_grad", M=8192, N=4096, gate=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_SIZE = {"f32": 4, "bf16": 2}


def draw(rng):
    while True:
        if rng.random() < 0.3:
            c = dict(_NORM, op=rng.choice(("norm", "norm_grad")), M=_log_int(rng, 1, 32768), N=_log_int(rng, 64, 16384),
                     x=rng.choice(("bf16", "f32")), y=rng.choice(("bf16", "f32")), h=rng.choice(("bf16", "f32")),
                     pre=rng.random() < 0.8, post=rng.random() < 0.8)
            if rng.random() < 0.6:
                c["N"] = max(64, c["N"] // 64 * 64)
            # no gate, one for every row, one per sample, one per row
            c["gate"] = rng.choice((0, c["M"], max(1, c["M"] // rng.randint(2, 9)), 1))
            if c["gate"]:
                c["M"] = c["M"] // c["gate"] * c["gate"]
            if not (c["pre"] or c["post"]) or c["M"] * c["N"] > 8192 * 4096:
                continue
            return c
        c = dict(_MM, op=rng.choice(("fwd", "fwd", "grad_x", "grad_w", "int8", "int8")), M=_log_int(rng, 1, 49152),
                 E=_log_int(rng, 1, 128), K=_log_int(rng, 64, 14336), N=_log_int(rng, 64, 14336),
                 w=rng.choice(("bf16", "bf16", "f32")), layout=rng.choice(("llama", "flux")),
                 skew=rng.choice(("none", "normal", "zipf")), tail=rng.choice((0, 0, 0, 77)),
                 pad=rng.choice((0, 0, 0, 8, 3)))
        if rng.random() < 0.6:
            c["K"], c["N"] = max(64, c["K"] // 64 * 64), max(64, c["N"] // 64 * 64)
        c["o"] = "f32" if c["w"] == "f32" else rng.choice(("bf16", "bf16", "f32"))
        if c["op"] == "int8":
            c["layout"], c["o"] = "llama", rng.choice(("bf16", "f32"))
        flops, wbytes = 2 * c["M"] * c["K"] * c["N"], c["E"] * c["K"] * c["N"] * _SIZE[c["w"]]
        if flops > (9.6e11 if c["w"] == "bf16" else 5e10) or wbytes > 9.5e8:
            continue
        return c


# ---- inputs --------------------------------------------------------------------

def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + part) & 0x7FFFFFFFFFFFFFFF)
    return g


_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rows(c, seed):
    """Rows of each group: M rows dealt to the E experts by their popularity."""
    rng = np.random.default_rng(int(seed) & 0x7FFFFFFFFFFFFFFF)
    p = {"none": np.ones(c["E"]), "normal": np.exp(rng.standard_normal(c["E"]) * 0.5),
         "zipf": rng.permutation(1.0 / np.arange(1, c["E"] + 1) ** 1.1)}[c["skew"]]
    return [int(v) for v in rng.multinomial(c["M"], p / p.sum())]


def _randn(g, rows, cols, scale, dtype, pad):
    t = torch.randn(rows, cols + pad, generator=g, device="cuda").mul_(scale)
    return t.to(dtype)[:, :cols]


def _weights(c, seed):
    """(E, out, in) or (E, in, out), N(0, 1 / K)."""
    g = _gen(seed, 1)
    shape = (c["N"], c["K"]) if c["layout"] == "llama" else (c["K"], c["N"])
    w = torch.empty(c["E"], *shape, device="cuda", dtype=_TYPE[c["w"]])
    for e in range(c["E"]):
        w[e] = torch.randn(*shape, generator=g, device="cuda").mul_(c["K"] ** -0.5)
    return w


def _matmul_inputs(c, seed):
    """x (M + tail, K) and dy (M + tail, N), the weights, the groups' rows."""
    g, dt, rows = _gen(seed, 0), _TYPE[c["w"]], c["M"] + c["tail"]
    x = dy = w = None
    if c["op"] in ("fwd", "grad_w", "int8"):
        x = _randn(g, rows, c["K"], 1.0, dt, c["pad"])
    if c["op"] in ("grad_x", "grad_w"):
        dy = _randn(g, rows, c["N"], 1.0, dt, c["pad"])
    if c["op"] != "grad_w":
        w = _weights(c, seed)
    return x, dy, w, _rows(c, seed)


def _int8_weights(w):
    """Codes and a scale per output channel, laid out once by the user."""
    q = torch.empty(w.shape, device="cuda", dtype=torch.int8)
    s = torch.empty(w.shape[:2], device="cuda")
    for e in range(w.shape[0]):
        f = w[e].float()
        most = f.abs().amax(dim=1, keepdim=True)
        s[e] = most[:, 0] / 127.0
        q[e] = torch.round(f * 127.0 / most).to(torch.int8)
    return q, s


def _norm_inputs(c, seed):
    g, M, N = _gen(seed, 0), c["M"], c["N"]
    new = lambda r, t: torch.randn(r, N, generator=g, device="cuda").to(t)
    s = dict(x=new(M, _TYPE[c["x"]]), y=new(M, _TYPE[c["y"]]).mul_(0.5), pre=None, post=None, gate=None)
    if c["pre"]:
        s["pre"] = 1.0 + 0.1 * new(1, torch.float32)[0]
    if c["post"]:
        s["post"] = 1.0 + 0.1 * new(1, torch.float32)[0]
    if c["gate"]:
        s["gate"] = new(M // c["gate"], _TYPE[c["x"]])
    if c["op"] == "norm_grad":
        s["dr"] = new(M, _TYPE[c["x"]])
        s["dh"] = new(M, _TYPE[c["h"]]) if c["pre"] else None
        # what a training step keeps of the forward pass
        f = _norm(s, torch.float32, _TYPE[c["x"]])
        s["r"], s["stats"] = f["r"].to(_TYPE[c["x"]]), torch.stack([f["iy"][:, 0], f["ir"][:, 0]], dim=1).contiguous()
    return s


def prepare(c, seed):
    if c["op"].startswith("norm"):
        return dict(case=c, **_norm_inputs(c, seed))
    x, dy, w, rows = _matmul_inputs(c, seed)
    offsets = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32, device="cuda")
    s = dict(case=c, x=x, dy=dy, rows=rows, offsets=offsets, w=w)
    if c["op"] == "int8":
        s["w"], s["ws"] = _int8_weights(w)
    cols = {"fwd": c["N"], "int8": c["N"], "grad_x": c["K"]}.get(c["op"])
    if cols is not None:  # rows behind the last group keep what the buffer held
        s["out"] = torch.zeros(c["M"] + c["tail"], cols, dtype=_TYPE[c["o"]], device="cuda")
    else:
        shape = (c["N"], c["K"]) if c["layout"] == "llama" else (c["K"], c["N"])
        s["out"] = torch.zeros(c["E"], *shape, dtype=_TYPE[c["o"]], device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------

def _groups(rows):
    at = 0
    for e, n in enumerate(rows):
        yield e, slice(at, at + n)
        at += n


def _rms(v, eps):
    return torch.rsqrt((v * v).mean(dim=1, keepdim=True) + eps)


def _norm(s, wide, rtype):
    """The forward pass in `wide`: r as the residual stream's type holds it."""
    w = lambda t: None if t is None else t.to(wide)
    x, y, gate = w(s["x"]), w(s["y"]), w(s["gate"])
    iy, z = torch.ones_like(y[:, :1]), y
    if s["post"] is not None:
        iy = _rms(y, _EPS)
        z = y * iy * w(s["post"])
    if gate is not None:
        z = z * gate.repeat_interleave(x.shape[0] // gate.shape[0], dim=0)
    r = (_ALPHA * x + _BETA * z).to(rtype).to(wide)
    ir = _rms(r, _EPS)
    return dict(r=r, iy=iy, ir=ir, h=r * ir * w(s["pre"]) if s["pre"] is not None else None)


def _norm_grad(s, r, iy, ir, wide):
    """dx, dy, dgate, dpost, dpre from dr and dh."""
    w = lambda t: t.to(wide)
    g, dpre, dpost, dgate = w(s["dr"]), None, None, None
    y, M = w(s["y"]), r.shape[0]
    if s["pre"] is not None:
        dh, rhat = w(s["dh"]), r * ir
        dpre = (dh * rhat).sum(dim=0)
        a = dh * w(s["pre"])
        g = g + ir * (a - rhat * (a * rhat).mean(dim=1, keepdim=True))
    u = _BETA * g
    yhat = y * iy if s["post"] is not None else y
    dz = u
    if s["gate"] is not None:
        G = s["gate"].shape[0]
        z = yhat * w(s["post"]) if s["post"] is not None else yhat
        dgate = (u * z).reshape(G, M // G, -1).sum(dim=1)
        dz = u * w(s["gate"]).repeat_interleave(M // G, dim=0)
    dy = dz
    if s["post"] is not None:
        dpost = (dz * yhat).sum(dim=0)
        a = dz * w(s["post"])
        dy = iy * (a - yhat * (a * yhat).mean(dim=1, keepdim=True))
    return dict(dx=_ALPHA * g, dy=dy, dgate=dgate, dpost=dpost, dpre=dpre)


def _norm_result(c, s, f):
    """Outputs in the order and types a caller gets them; None left out."""
    xt, yt, ht, f32 = _TYPE[c["x"]], _TYPE[c["y"]], _TYPE[c["h"]], torch.float32
    types = dict(r=xt, h=ht) if c["op"] == "norm" else dict(dx=xt, dy=yt, dgate=f32, dpost=f32, dpre=f32)
    return [f[k].to(t) for k, t in types.items() if f[k] is not None]


def _run_own(s):
    import mixtureofexperts_amd as moe
    from mixtureofexperts_amd import _lib

    c = s["case"]
    if c["op"] == "norm":
        r, h, _ = moe.block_norm(s["x"], s["y"], pre_weight=s["pre"], post_weight=s["post"], gate=s["gate"],
                                 alpha=_ALPHA, beta=_BETA, eps=_EPS, h_dtype=_TYPE[c["h"]])
        return [t for t in (r, h) if t is not None]
    if c["op"] == "norm_grad":
        grads = moe.block_norm_grad(s["dr"], s["dh"], s["r"], s["y"], s["stats"], pre_weight=s["pre"],
                                    post_weight=s["post"], gate=s["gate"], alpha=_ALPHA, beta=_BETA)
        return [t for t in grads if t is not None]
    layout = _lib.MOE_LAYOUT_LLAMA_IN_OUT if c["layout"] == "llama" else _lib.MOE_LAYOUT_FLUX_OUT_IN
    if c["op"] == "fwd":
        return [moe.grouped_matmul(s["x"], s["w"], s["offsets"], layout=layout, out=s["out"])]
    if c["op"] == "grad_x":
        return [moe.grouped_matmul_grad_x(s["dy"], s["w"], s["offsets"], layout=layout, out=s["out"])]
    if c["op"] == "grad_w":
        return [moe.grouped_matmul_grad_w(s["x"], s["dy"], s["offsets"], layout=layout, out=s["out"])]
    return [moe.int8_matmul(s["x"], s["w"], s["ws"], s["offsets"], out=s["out"])]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "norm":
        return _norm_result(c, s, _norm(s, torch.float32, _TYPE[c["x"]]))
    if c["op"] == "norm_grad":
        return _norm_result(c, s, _norm_grad(s, s["r"].float(), s["stats"][:, :1], s["stats"][:, 1:], torch.float32))
    out, flux = s["out"], c["layout"] == "flux"
    if c["op"] == "int8":
        x = s["x"].float()
        most = x.abs().amax(dim=1, keepdim=True)
        sx = most / 127.0
        # 127 x first: a code's border, an odd multiple of most / 254, is then met exactly
        q = torch.where(most > 0, torch.round(x * 127.0 / most), torch.zeros_like(x))
    for e, g in _groups(s["rows"]):
        if g.start == g.stop and c["op"] != "grad_w":
            continue
        if c["op"] == "fwd":
            w = s["w"][e].float()
            out[g] = s["x"][g].float() @ (w if flux else w.t())
        elif c["op"] == "grad_x":
            w = s["w"][e].float()
            out[g] = s["dy"][g].float() @ (w.t() if flux else w)
        elif c["op"] == "grad_w":
            a, b = (s["x"], s["dy"]) if flux else (s["dy"], s["x"])
            out[e] = a[g].float().t() @ b[g].float()
        else:
            out[g] = (q[g] @ s["w"][e].float().t()) * sx[g] * s["ws"][e]
    return [out]


# ---- what a pass cannot do without ----------------------------------------------

def work(c):
    if c["op"].startswith("norm"):
        M, N = c["M"], c["N"]
        gates = M // c["gate"] if c["gate"] else 0
        x, y, h = _SIZE[c["x"]], _SIZE[c["y"]], _SIZE[c["h"]] * c["pre"]
        small = 4 * N * (c["pre"] + c["post"])
        if c["op"] == "norm":
            return {"bytes": M * N * (2 * x + y + h) + small + gates * N * x, "flops": 12.0 * M * N}
        return {"bytes": M * N * (3 * x + 2 * y + h) + 2 * small + gates * N * (x + 4) + 8 * M, "flops": 30.0 * M * N}
    M, E, K, N = c["M"], c["E"], c["K"], c["N"]
    hit = E * (1 - (1 - 1 / E) ** M)  # groups that hold a row, at an even load
    es, eo = _SIZE[c["w"]], _SIZE[c["o"]]
    flops = 2.0 * M * K * N
    if c["op"] == "grad_w":
        return {"bytes": M * (K + N) * es + E * K * N * eo, "flops": flops}
    if c["op"] == "int8":
        return {"bytes": M * (K * es + N * eo) + hit * (K * N + 4 * N), "flops": flops}
    wide, narrow = (N, K) if c["op"] == "fwd" else (K, N)
    return {"bytes": M * (narrow * es + wide * eo) + hit * K * N * es, "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------

def exact(c, seed):
    if c["op"].startswith("norm"):
        return _exact_norm(c, _norm_inputs(c, seed))
    x, dy, w, rows = _matmul_inputs(c, seed)
    total, f64 = c["M"] + c["tail"], torch.float64
    bounds = np.concatenate([[0], np.cumsum(rows)])
    if c["op"] == "grad_w":
        left, right = (dy, x) if c["layout"] == "llama" else (x, dy)
        dw = torch.zeros(c["E"], left.shape[1], right.shape[1], dtype=f64, device="cuda")
        for e in range(c["E"]):
            lo, hi = int(bounds[e]), int(bounds[e + 1])
            if hi > lo:
                dw[e] = torch.mm(left[lo:hi].to(f64).t().contiguous(), right[lo:hi].to(f64))
        return [dw]
    src = dy if c["op"] == "grad_x" else x
    # the matrix a row is multiplied with from the right: (columns of src, columns of the result)
    turn = (c["op"] == "grad_x") == (c["layout"] == "flux")
    if c["op"] == "int8":
        w, ws = _int8_weights(w)
        amax = src.abs().amax(dim=1).to(f64)
        sx = (amax / 127.0).to(torch.float32).to(f64)  # the scale is held in 32 bits
    out = torch.zeros(total, c["K"] if c["op"] == "grad_x" else c["N"], dtype=f64, device="cuda")
    for e in range(c["E"]):
        lo, hi = int(bounds[e]), int(bounds[e + 1])
        if hi == lo:
            continue
        a, b = src[lo:hi].to(f64), w[e].to(f64)
        if turn:
            b = b.t().contiguous()
        if c["op"] == "int8":
            safe = torch.where(amax[lo:hi] > 0, amax[lo:hi], torch.ones_like(amax[lo:hi]))
            a = torch.round(127.0 * a / safe[:, None])
            out[lo:hi] = torch.mm(a, b) * sx[lo:hi, None] * ws[e].to(f64)[None, :]
        else:
            out[lo:hi] = torch.mm(a, b)
    return [out]


def _exact_norm(c, s):
    f64 = torch.float64
    d = {k: (v.to(f64) if v is not None and k in ("x", "y", "pre", "post", "gate", "dr", "dh", "r") else v)
         for k, v in s.items()}
    M, N = c["M"], c["N"]
    ones = torch.ones(1, N, dtype=f64, device="cuda")
    post = d["post"] if c["post"] else ones
    pre = d["pre"] if c["pre"] else None
    gate = ones if d["gate"] is None else d["gate"].unsqueeze(1).expand(-1, c["gate"], -1).reshape(M, N)
    ny = ((d["y"] ** 2).sum(1, keepdim=True) / N + _EPS) ** -0.5 if c["post"] else torch.ones(M, 1, dtype=f64, device="cuda")
    yhat = d["y"] * ny
    if c["op"] == "norm":
        r = _ALPHA * d["x"] + _BETA * gate * yhat * post
        if pre is None:
            return [r]
        held = r.to(_TYPE[c["x"]]).to(f64)  # h is the norm of the stream as it is stored
        return [r, held * ((held ** 2).sum(1, keepdim=True) / N + _EPS) ** -0.5 * pre]
    total, dpre = d["dr"], None
    if pre is not None:
        nr = ((d["r"] ** 2).sum(1, keepdim=True) / N + _EPS) ** -0.5
        rhat = d["r"] * nr
        dpre = (d["dh"] * rhat).sum(0)
        t = d["dh"] * pre
        total = total + nr * t - nr * rhat * ((t * rhat).sum(1, keepdim=True) / N)
    out = [_ALPHA * total]
    dz = _BETA * total * gate
    if c["post"]:
        t = dz * post
        out.append(ny * t - ny * yhat * ((t * yhat).sum(1, keepdim=True) / N))
    else:
        out.append(dz)
    if c["gate"]:
        out.append((_BETA * total * yhat * post).reshape(M // c["gate"], c["gate"], N).sum(1))
    if c["post"]:
        out.append((dz * yhat).sum(0))
    if dpre is not None:
        out.append(dpre)
    return out
