"""The gate's own values in gated_matmul_grad at the infinities."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

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
