"""The operators of ops.py together, as a program uses them: a training step
through an MoE FFN block (norm, routed products, post norm with gate and
residual, all gradients) against float64 autograd on the CPU; the same block
served with int8 experts; and moe_block_forward, the layer between its norms.

Tolerances are relative to the norm of each result.  fp32: a path crosses at
most six products of up to 256 terms, each off by at most 256 * 2^-24 of its
magnitudes' sum, which is up to sqrt(256) times its norm for random terms:
6 * 256 * 16 * 2^-24 < 1.5e-3.  bf16: at most ten roundings to bf16 on a path,
each at most 2^-8 of its value: 4e-2.  int8: the reference is the same
arithmetic on the same codes, so only the fp32 and bf16 roundings count."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _rel(got, ref):
    got, ref = got.detach().cpu().double(), ref.detach().double()
    return float((got - ref).norm() / ref.norm())


def _problem(dtype, seed, T=150, D=96, H=256, E=6, k=2):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    p = dict(x=rnd(T, D), w1=rnd(E, H, D) * D**-0.5, w3=rnd(E, H, D) * D**-0.5, w2=rnd(E, D, H) * H**-0.5,
             pre=1 + 0.1 * rnd(D), post=1 + 0.1 * rnd(D), nxt=1 + 0.1 * rnd(D), gate=rnd(3, D))
    low = ("x", "w1", "w2", "w3", "gate")
    p = {n: (t.to(dtype) if n in low else t) for n, t in p.items()}
    # routing is given (the layer's own); expert 4 gets no token
    logits = rnd(T, E)
    logits[:, 4] = -1e9
    v, i = torch.topk(torch.softmax(logits, 1), k, dim=1)
    p["gates"], p["idx"] = v / v.sum(1, keepdim=True), i
    flat = i.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    p["token"] = order // k
    p["weight"] = p["gates"].reshape(-1)[order]
    p["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(flat, minlength=E).cumsum(0)]).int()
    return p


ALPHA, BETA = 0.9, 1.1


def _reference(p, leaves):
    """(r, n) in float64 with autograd."""
    q = {n: leaves.get(n, t.double() if t.is_floating_point() else t) for n, t in p.items()}
    rms = lambda v: v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5)
    h = rms(q["x"]) * q["pre"]
    rows, out = h[q["token"]], []
    o = p["offsets"].tolist()
    for e in range(len(o) - 1):
        s = rows[o[e]:o[e + 1]]
        out.append((torch.nn.functional.silu(s @ q["w1"][e].t()) * (s @ q["w3"][e].t())) @ q["w2"][e].t())
    y = torch.zeros_like(h).index_add(0, q["token"], torch.cat(out) * q["weight"][:, None])
    z = rms(y) * q["post"] * q["gate"].repeat_interleave(h.shape[0] // 3, 0)
    r = ALPHA * q["x"] + BETA * z
    return r, rms(r) * q["nxt"]


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1.5e-3), (torch.bfloat16, 4e-2)])
def test_training_step(moe, dtype, tol):
    print(f"block training step {dtype}", flush=True)
    p = _problem(dtype, 1)
    d = {n: t.cuda() for n, t in p.items()}
    T = d["x"].shape[0]
    # forward
    _, h, st0 = moe.block_norm(d["x"], pre_weight=d["pre"])
    rows = h[d["token"]]
    a = moe.grouped_matmul(rows, d["w1"], d["offsets"])
    b = moe.grouped_matmul(rows, d["w3"], d["offsets"])
    s = torch.sigmoid(a.float())
    act = (a.float() * s * b.float()).to(dtype)
    yr = moe.grouped_matmul(act, d["w2"], d["offsets"], out_dtype=torch.float32)
    y = torch.zeros(T, yr.shape[1], device="cuda").index_add(0, d["token"], yr * d["weight"][:, None])
    kw = dict(pre_weight=d["nxt"], post_weight=d["post"], gate=d["gate"], alpha=ALPHA, beta=BETA)
    r, n, st1 = moe.block_norm(d["x"], y, **kw)
    # backward
    g = torch.Generator().manual_seed(2)
    dr, dn = (torch.randn(r.shape, generator=g).to(dtype) for _ in range(2))
    dx, dy, dgate, dpost, dnxt = moe.block_norm_grad(dr.cuda(), dn.cuda(), r, y, st1, **kw)
    dyr = (dy[d["token"]] * d["weight"][:, None]).to(dtype)
    dw2 = moe.grouped_matmul_grad_w(act, dyr, d["offsets"], out_dtype=torch.float32)
    dact = moe.grouped_matmul_grad_x(dyr, d["w2"], d["offsets"]).float()
    da = (dact * b.float() * (s + a.float() * s * (1 - s))).to(dtype)
    db = (dact * a.float() * s).to(dtype)
    dw1 = moe.grouped_matmul_grad_w(rows, da, d["offsets"], out_dtype=torch.float32)
    dw3 = moe.grouped_matmul_grad_w(rows, db, d["offsets"], out_dtype=torch.float32)
    drows = moe.grouped_matmul_grad_x(da, d["w1"], d["offsets"], out_dtype=torch.float32)
    drows += moe.grouped_matmul_grad_x(db, d["w3"], d["offsets"], out_dtype=torch.float32)
    dh = torch.zeros(T, h.shape[1], device="cuda").index_add(0, d["token"], drows)
    dx0, _, _, _, dpre = moe.block_norm_grad(None, dh, d["x"], None, st0, pre_weight=d["pre"])
    total = dx.float() + dx0.float()

    leaves = {m: p[m].double().requires_grad_() for m in ("x", "w1", "w2", "w3", "pre", "post", "nxt", "gate")}
    R, N = _reference(p, leaves)
    (R * dr.double()).sum().backward(retain_graph=True)
    (N * dn.double()).sum().backward()
    assert _rel(r, R) <= tol and _rel(n, N) <= tol
    for name, got in (("x", total), ("w1", dw1), ("w2", dw2), ("w3", dw3), ("pre", dpre), ("post", dpost), ("nxt", dnxt),
                      ("gate", dgate)):
        assert _rel(got, leaves[name].grad) <= tol, (name, _rel(got, leaves[name].grad))
    assert (dw1[4] == 0).all() and (dw2[4] == 0).all()  # no token chose expert 4


@pytest.mark.parametrize("T", [1, 7, 150])
def test_int8_serving(moe, T):
    print(f"block int8 serving T={T}", flush=True)
    p = _problem(torch.bfloat16, 3, T=150)
    keep = p["token"] < T
    off = p["offsets"].tolist()
    rows_of = [int(keep[off[e]:off[e + 1]].sum()) for e in range(6)]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(rows_of)]), dtype=torch.int32, device="cuda")
    token, weight = p["token"][keep].cuda(), p["weight"][keep].cuda()
    d = {n: t.cuda() for n, t in p.items()}
    x = d["x"][:T].contiguous()
    w = {n: moe.quantize_int8(d[n]) for n in ("w1", "w2", "w3")}
    _, h, _ = moe.block_norm(x, pre_weight=d["pre"])
    rows = h[token]
    q, s = moe.quantize_int8(rows)
    a = moe.int8_matmul(q, *w["w1"], offsets, x_scale=s, out_dtype=torch.float32)
    b = moe.int8_matmul(rows, *w["w3"], offsets, out_dtype=torch.float32)
    act = (torch.nn.functional.silu(a) * b).to(torch.bfloat16)
    yr = moe.int8_matmul(act, *w["w2"], offsets, out_dtype=torch.float32)
    y = torch.zeros(T, yr.shape[1], device="cuda").index_add(0, token, yr * weight[:, None])
    r, n, _ = moe.block_norm(x, y, pre_weight=d["nxt"], post_weight=d["post"])

    def dense(v, name):  # the codes' values, float64 on the CPU
        vq, vs = (t.cpu().double() for t in moe.quantize_int8(v))
        wq, ws = (t.cpu().double() for t in w[name])
        o, out = offsets.tolist(), []
        for e in range(6):
            out.append((vq[o[e]:o[e + 1]] @ wq[e].t()) * vs[o[e]:o[e + 1], None] * ws[e])
        return torch.cat(out)

    assert _rel(a, dense(rows, "w1")) <= 1e-6 and _rel(b, dense(rows, "w3")) <= 1e-6
    assert _rel(yr, dense(act, "w2")) <= 1e-6
    # against the float weights: a code is off by at most half a step of 1/127 of
    # its row's largest; three quantised products in a row, a few percent each
    leaves = {}
    P = dict(p, x=p["x"][:T], token=p["token"][keep], weight=p["weight"][keep], offsets=offsets.cpu())
    rms = lambda v: v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5)
    H = (rms(P["x"].double()) * P["pre"].double())[P["token"]]
    o, out = P["offsets"].tolist(), []
    for e in range(6):
        v = H[o[e]:o[e + 1]]
        f = lambda m: P[m][e].double().t()
        out.append((torch.nn.functional.silu(v @ f("w1")) * (v @ f("w3"))) @ f("w2"))
    assert _rel(yr, torch.cat(out)) <= 0.1


@pytest.mark.parametrize("weight_dtype,xt", [("f32", torch.float32), ("bf16", torch.bfloat16), ("bf16", torch.float32)])
def test_block_forward(moe, weight_dtype, xt):
    print(f"moe_block_forward {weight_dtype} {xt}", flush=True)
    rng = np.random.default_rng(4)
    cfg = moe.MoEConfig(num_experts=8, expert_type="gated", input_dim=128, hidden_dim=256, output_dim=128,
                        activation=moe.silu, gate_type=moe.TopKGating(2), weight_dtype=weight_dtype, max_tokens=128)
    layer = moe.MoELayer(cfg, rng=rng)
    x = torch.from_numpy(rng.standard_normal((60, 128)).astype(np.float32)).to(xt).cuda()
    pre, post, nxt = (torch.from_numpy((1 + 0.1 * rng.standard_normal(128)).astype(np.float32)).cuda() for _ in range(3))
    gate = torch.from_numpy(rng.standard_normal((2, 128)).astype(np.float32)).cuda()
    rms = lambda v: v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5)
    for decode in (False, True):
        r, n, loss = moe.moe_block_forward(layer, x, pre_weight=pre, post_weight=post, gate=gate, next_weight=nxt,
                                           alpha=ALPHA, beta=BETA, training=not decode, decode=decode)
        _, h, _ = moe.block_norm(x, pre_weight=pre, h_dtype=torch.bfloat16 if (
            weight_dtype == "bf16" and xt == torch.bfloat16 and not decode) else torch.float32)
        if decode:
            y = torch.from_numpy(np.ascontiguousarray(moe.moe_ffn_forward(layer, h.cpu().numpy().T)[0].T))
        else:
            out, want = layer(h.float().cpu().numpy().T, training=True)
            y = torch.from_numpy(np.ascontiguousarray(out.T))
            assert abs(float(loss) - float(want)) <= 1e-5 * max(1.0, abs(float(want)))
        y = y.double()
        R = ALPHA * x.cpu().double() + BETA * gate.cpu().double().repeat_interleave(30, 0) * rms(y) * post.cpu().double()
        # r and n in x's type: one rounding each, the layer's own output the same
        tol = 2.0**-8 if xt == torch.bfloat16 else 1e-5
        assert r.dtype == xt and _rel(r, R) <= tol
        assert _rel(n, rms(r.cpu().double()) * nxt.cpu().double()) <= tol
    r, n, loss = moe.moe_block_forward(layer, x, pre_weight=pre)
    assert n is None and float(loss) == 0.0
    r0, _, _ = moe.moe_block_forward(layer, x[:0], pre_weight=pre)
    assert r0.shape == (0, 128)
    for bad, msg in ((dict(pre_weight=None), "pre_weight"), (dict(pre_weight=pre, gate=gate[:, :5]), "gate")):
        with pytest.raises(moe.MoeError, match=msg):
            moe.moe_block_forward(layer, x, **bad)
    with pytest.raises(moe.MoeError):
        moe.moe_block_forward(layer, x[:, :64], pre_weight=pre)
    layer.close()


def test_block_forward_refuses_host_gates(moe):
    cfg = moe.MoEConfig(num_experts=4, expert_type="gated", input_dim=32, hidden_dim=64, output_dim=32,
                        activation=moe.silu, gate_type=moe.RandomGating(2), max_tokens=8)
    with pytest.raises(moe.MoeError, match="host"):
        moe.moe_block_forward(moe.MoELayer(cfg), torch.zeros(2, 32, device="cuda"), pre_weight=torch.ones(32, device="cuda"))


@pytest.mark.parametrize("decode", [False, True])
def test_block_forward_on_streams(moe, decode):
    # the same bits on torch's null stream and on another one, in turn on one layer;
    # a capture is refused (the layer's calls order themselves by events)
    rng = np.random.default_rng(16)
    cfg = moe.MoEConfig(num_experts=8, expert_type="gated", input_dim=128, hidden_dim=256, output_dim=128,
                        activation=moe.silu, gate_type=moe.TopKGating(2), weight_dtype="bf16", max_tokens=64)
    layer = moe.MoELayer(cfg, rng=rng)
    T = 3 if decode else 50
    xs = [torch.from_numpy(rng.standard_normal((T, 128)).astype(np.float32)).cuda() for _ in range(3)]
    pre, post = (torch.ones(128, device="cuda") for _ in range(2))
    step = lambda x: moe.moe_block_forward(layer, x, pre_weight=pre, post_weight=post, next_weight=pre, decode=decode)[:2]
    want = []
    for x in xs:
        want.append(step(x))
        torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    for turn in range(4):
        for i, x in enumerate(xs):
            if (turn + i) % 2:
                with torch.cuda.stream(side):
                    got.append((i, step(x)))
            else:
                got.append((i, step(x)))
    torch.cuda.synchronize()
    for i, res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want[i])), i
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(moe.MoeError, match="captured"):
            step(xs[0])
        y = xs[0] + 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, xs[0] + 1)
    layer.close()


def test_block_forward_refuses_too_many_tokens(moe):
    cfg = moe.MoEConfig(num_experts=4, expert_type="gated", input_dim=32, hidden_dim=64, output_dim=32,
                        activation=moe.silu, gate_type=moe.TopKGating(2), max_tokens=8)
    layer = moe.MoELayer(cfg)
    pre = torch.ones(32, device="cuda")
    for decode in (False, True):
        with pytest.raises(moe.MoeError):
            moe.moe_block_forward(layer, torch.zeros(4096, 32, device="cuda"), pre_weight=pre, decode=decode)
    r, _, _ = moe.moe_block_forward(layer, torch.ones(8, 32, device="cuda"), pre_weight=pre)
    assert torch.isfinite(r).all()
    with pytest.raises(moe.MoeError, match="GPU memory"):
        moe.moe_block_forward(layer, torch.ones(8, 32), pre_weight=pre)
    layer.close()


@pytest.mark.parametrize("T", [1, 7, 150])
def test_int8_serving_to_the_end(moe, T):
    # the same block's last steps: the experts' rows gathered by token, the norm of
    # their sum with the residual, and the norm of the stream
    print(f"block int8 serving to the end T={T}", flush=True)
    p = _problem(torch.bfloat16, 3, T=150)
    keep = p["token"] < T
    off = p["offsets"].tolist()
    offsets = np.concatenate([[0], np.cumsum([int(keep[off[e]:off[e + 1]].sum()) for e in range(6)])]).tolist()
    token, weight = p["token"][keep], p["weight"][keep]
    d = {n: t.cuda() for n, t in p.items()}
    x = d["x"][:T].contiguous()
    w2, s2 = moe.quantize_int8(d["w2"])
    rng = np.random.default_rng(T)
    act = torch.from_numpy(rng.standard_normal((len(token), 256))).to(torch.bfloat16).cuda()
    yr = moe.int8_matmul(act, w2, s2, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    y = torch.zeros(T, yr.shape[1], device="cuda").index_add(0, token.cuda(), yr * weight.cuda()[:, None])
    r, n, _ = moe.block_norm(x, y, pre_weight=d["nxt"], post_weight=d["post"])
    # float64 on the CPU, from the codes' values
    q, s = (t.cpu().double() for t in moe.quantize_int8(act))
    wq, ws = w2.cpu().double(), s2.cpu().double()
    o = offsets
    rows = torch.cat([(q[o[e]:o[e + 1]] @ wq[e].t()) * s[o[e]:o[e + 1], None] * ws[e] for e in range(6)])
    Y = torch.zeros(T, rows.shape[1], dtype=torch.float64).index_add(0, token, rows * weight.double()[:, None])
    rms = lambda v: v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5)
    X, Z = p["x"][:T].double(), rms(Y) * p["post"].double()
    # r: fp32 steps (1e-5 of the terms, which may cancel), then one rounding to bf16;
    # n: the norm of r as it is stored, the same
    assert ((r.cpu().double() - (X + Z)).abs() <= 2.0**-8 * (X + Z).abs() + 1e-5 * (X.abs() + Z.abs())).all()
    N = rms(r.cpu().double()) * p["nxt"].double()
    assert ((n.cpu().double() - N).abs() <= (2.0**-8 + 1e-5) * N.abs()).all()
