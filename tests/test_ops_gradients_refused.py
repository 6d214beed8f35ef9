"""Tensors that torch would differentiate: the operators record nothing, so they
refuse them instead of cutting the graph, and tell torch what they write to."""
import pytest

torch = pytest.importorskip("torch")


def _calls(moe, mark, dev):
    """(call, name of the marked operand) for every tensor operand of every
    function; mark(t) makes t one that torch would differentiate."""
    z = lambda *s: torch.zeros(*s, device=dev)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device=dev)
    w, ws = (2, 6, 8), (2, 6)
    return [
        ("x", lambda: moe.grouped_matmul(mark(z(4, 8)), z(*w), off)),
        ("w", lambda: moe.grouped_matmul(z(4, 8), mark(z(*w)), off)),
        ("out", lambda: moe.grouped_matmul(z(4, 8), z(*w), off, out=mark(z(4, 6)))),
        ("dy", lambda: moe.grouped_matmul_grad_x(mark(z(4, 6)), z(*w), off)),
        ("w", lambda: moe.grouped_matmul_grad_x(z(4, 6), mark(z(*w)), off)),
        ("out", lambda: moe.grouped_matmul_grad_x(z(4, 6), z(*w), off, out=mark(z(4, 8)))),
        ("x", lambda: moe.grouped_matmul_grad_w(mark(z(4, 8)), z(4, 6), off)),
        ("dy", lambda: moe.grouped_matmul_grad_w(z(4, 8), mark(z(4, 6)), off)),
        ("out", lambda: moe.grouped_matmul_grad_w(z(4, 8), z(4, 6), off, out=mark(z(*w)))),
        ("x", lambda: moe.quantize_int8(mark(z(4, 8)))),
        ("x", lambda: moe.int8_matmul(mark(z(4, 8)), i8(*w), z(*ws), off)),
        ("w_scale", lambda: moe.int8_matmul(z(4, 8), i8(*w), mark(z(*ws)), off)),
        ("x_scale", lambda: moe.int8_matmul(i8(4, 8), i8(*w), z(*ws), off, x_scale=mark(z(4)))),
        ("out", lambda: moe.int8_matmul(z(4, 8), i8(*w), z(*ws), off, out=mark(z(4, 6)))),
        ("x", lambda: moe.block_norm(mark(z(4, 8)), pre_weight=z(8))),
        ("y", lambda: moe.block_norm(z(4, 8), mark(z(4, 8)), pre_weight=z(8))),
        ("pre_weight", lambda: moe.block_norm(z(4, 8), pre_weight=mark(z(8)))),
        ("post_weight", lambda: moe.block_norm(z(4, 8), z(4, 8), post_weight=mark(z(8)))),
        ("gate", lambda: moe.block_norm(z(4, 8), z(4, 8), gate=mark(z(8)))),
        ("dr", lambda: moe.block_norm_grad(mark(z(4, 8)), None, z(4, 8), z(4, 8))),
        ("dh", lambda: moe.block_norm_grad(None, mark(z(4, 8)), z(4, 8), None, z(4, 2), pre_weight=z(8))),
        ("r", lambda: moe.block_norm_grad(z(4, 8), None, mark(z(4, 8)), z(4, 8))),
        ("y", lambda: moe.block_norm_grad(z(4, 8), None, z(4, 8), mark(z(4, 8)))),
        ("stats", lambda: moe.block_norm_grad(None, z(4, 8), z(4, 8), None, mark(z(4, 2)), pre_weight=z(8))),
        ("pre_weight", lambda: moe.block_norm_grad(None, z(4, 8), z(4, 8), None, z(4, 2), pre_weight=mark(z(8)))),
        ("gate", lambda: moe.block_norm_grad(z(4, 8), None, z(4, 8), z(4, 8), gate=mark(z(8)))),
    ]


def _tangent(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


def _refused(moe, dev):
    for name, call in _calls(moe, lambda t: t.requires_grad_(), dev):
        with pytest.raises(moe.MoeError, match=f"{name} requires a gradient"):
            call()
    with torch.autograd.forward_ad.dual_level():
        for name, call in _calls(moe, _tangent, dev):
            with pytest.raises(moe.MoeError, match=f"{name} carries a tangent"):
                call()


def test_refused_on_the_host(moe):
    # before anything else is looked at, so the CPU shows it too
    _refused(moe, "cpu")


def _layer(moe):
    cfg = moe.MoEConfig(num_experts=4, expert_type="gated", input_dim=32, hidden_dim=64, output_dim=32,
                        activation=moe.silu, gate_type=moe.TopKGating(2), max_tokens=8)
    return moe.MoELayer(cfg)


@pytest.mark.parametrize("name", ["x", "pre_weight", "post_weight", "gate", "next_weight"])
def test_block_refused_on_the_host(moe, name):
    # all five are looked at before the first norm runs
    a = dict(x=torch.zeros(2, 32), pre_weight=torch.ones(32), post_weight=torch.ones(32), gate=torch.ones(32),
             next_weight=torch.ones(32))
    a[name].requires_grad_()
    with pytest.raises(moe.MoeError, match=f"{name} requires a gradient"):
        moe.moe_block_forward(_layer(moe), a.pop("x"), **a)


@pytest.mark.gpu
def test_refused(moe):
    _refused(moe, "cuda")


@pytest.mark.gpu
def test_taken_where_nothing_is_recorded(moe):
    # torch.no_grad(), a tensor without the mark, and the forward and backward of
    # an autograd.Function: the way to train with these calls
    off = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    w = torch.randn(2, 6, 8, device="cuda", requires_grad=True)
    with torch.no_grad():
        want = moe.grouped_matmul(x, w, off)
    assert not want.requires_grad and torch.equal(want, moe.grouped_matmul(x.detach(), w.detach(), off))
    with torch.inference_mode():
        out = torch.empty(4, 6, device="cuda")
        assert torch.equal(moe.grouped_matmul(x, w, off, out=out), want)

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w)
            return moe.grouped_matmul(x, w, off)

        @staticmethod
        def backward(ctx, dy):
            x, w = ctx.saved_tensors
            return moe.grouped_matmul_grad_x(dy, w, off), moe.grouped_matmul_grad_w(x, dy, off)

    y = Product.apply(x, w)
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(y.detach(), want)
    assert torch.equal(x.grad, moe.grouped_matmul_grad_x(dy, w.detach(), off))
    assert torch.equal(w.grad, moe.grouped_matmul_grad_w(x.detach(), dy, off))


@pytest.mark.gpu
def test_written_results_are_seen_by_autograd(moe):
    # a tensor that a backward pass still needs, written by a call: torch notices
    off = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(2, 6, 8, device="cuda")
    q, s = moe.quantize_int8(w)
    dy = torch.randn(4, 6, device="cuda")
    for out, call in ((torch.zeros(4, 6, device="cuda"), lambda o: moe.grouped_matmul(x, w, off, out=o)),
                      (torch.zeros(4, 8, device="cuda"), lambda o: moe.grouped_matmul_grad_x(dy, w, off, out=o)),
                      (torch.zeros(2, 6, 8, device="cuda"), lambda o: moe.grouped_matmul_grad_w(x, dy, off, out=o)),
                      (torch.zeros(4, 6, device="cuda"), lambda o: moe.int8_matmul(x, q, s, off, out=o))):
        leaf = torch.ones_like(out, requires_grad=True)
        y = (leaf * out).sum()
        before = out._version
        call(out)
        assert out._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
