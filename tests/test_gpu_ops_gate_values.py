"""The gate's own values in gated_matmul and gated_matmul_grad: at the infinities, and how
near a float32 result of bfloat16 operands is."""
import numpy as np
import pytest

from op_kernels import kernels_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FLUX, LLAMA = 0, 1
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("down", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "identity"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_slope_at_infinities(moe, dtype, act, down):
    # what the formulas give: at -infinity silu and gelu are -inf * 0, NaN, as their slopes
    # are; at infinity the slope is 1
    inf = float("inf")
    a = torch.tensor([[-inf, inf, 1.0, float("nan")]], device="cuda", dtype=DT[dtype]).repeat(5, 1)
    dy, b = torch.ones_like(a), torch.full_like(a, 2.0)
    w2 = torch.eye(4, device="cuda", dtype=DT[dtype])[None].contiguous() if down else None
    da, db, h = (t.double().cpu() for t in moe.gated_matmul_grad(dy, a, b, w2, activation=getattr(moe, act)))
    low = {"relu": 0.0, "identity": 2.0}.get(act, float("nan"))
    for r in range(5):
        for t, ref in ((da, low), (db, -inf if act == "identity" else low), (h, -inf if act == "identity" else low)):
            assert torch.isnan(t[r, 0]) if np.isnan(ref) else t[r, 0] == ref, (act, t[r])
        assert da[r, 1] == 2.0 and db[r, 1] == inf and h[r, 1] == inf
        assert torch.isnan(db[r, 3]) and torch.isnan(h[r, 3])
        assert torch.isnan(da[r, 3]) or act in ("relu", "identity")


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_fp32_results_are_fp32_gates(moe, dtype, act, layout):
    """a = x and b = 1 exactly, so that h is the gate.  e^-z is off by 2^-23 of itself and
    by z's own error, 1 + e^-z, the division and the product with a by 2^-24 each: 5 2^-24
    (silu, z = a).  gelu's z: its two constants, two products (a a is exact for eight bits),
    the sum and the last product, 6 2^-24 of z, that many |z| times of e^-z.  With the terms
    of second order 6 2^-24 and (6 + 6 |z|) 2^-24."""
    # streamed; 64, 128 and 256-row tiles; k split over streams and over tiles
    for M, K, H, rows in ((3, 8, 24, None), (100, 8, 24, 64), (1600, 8, 1024, 128), (9000, 8, 2048, 256), (2, 8192, 16, None),
                          (70, 5440, 64, 64)):
        print(f"gate values {dtype} {act} layout={layout} M={M} K={K} H={H}", flush=True)
        v = torch.linspace(-80, 30, M) if act == "silu" else torch.linspace(-8, 6, M)
        x = torch.zeros(M, K, dtype=DT[dtype])
        x[:, 0], x[:, 1] = v.to(torch.bfloat16).to(DT[dtype]), 1
        w1, w3 = (torch.zeros(H, K, dtype=DT[dtype]) for _ in range(2))
        w1[:, 0], w3[:, 1] = 1, 1
        w1, w3 = (w if layout == LLAMA else w.t().contiguous() for w in (w1, w3))
        x, w1, w3, res = x.cuda(), w1.cuda(), w3.cuda(), []
        names = kernels_of(lambda: res.append(moe.gated_matmul(x, w1, w3, activation=getattr(moe, act), layout=layout,
                                                               out_dtype=torch.float32)))
        if dtype == "bf16" and rows in (128, 256):
            assert int(names["op_gated_kernel"][3]) == rows
        a = x[:, 0].double()
        z = a if act == "silu" else 2 * np.sqrt(2 / np.pi) * (a + 0.044715 * a**3)
        ref = a / (1 + torch.exp(-z))
        tol = (6 + (6 * z.abs() if act == "gelu" else 0)) * 2.0**-24 * ref.abs() + 2.0**-149
        bad = ~((res[0].double() - ref[:, None]).abs() <= tol[:, None])
        assert not bad.any(), (M, K, H, int(bad.sum()), ((res[0].double() - ref[:, None]).abs() / ref[:, None].abs()).nan_to_num().max().item() * 2**24)
