"""What moe_fp8_matmul_exact_async refuses: all that moe_fp8_matmul_async does, under its
own name.  Refused on the host: the pointers are never read."""
import pytest

from test_ops_fp8_refusals import FP8, INT8, MM, P, _refused


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "groups"), (dict(offsets=None), "offsets"), (dict(x_dtype=INT8), "x_dtype"), (dict(y_dtype=FP8), "result"),
    (dict(ldw=63), "row stride"), (dict(w_stride=64 * 32 - 1), "w_stride"), (dict(w_scale=None), "null"),
    (dict(x_dtype=FP8), "x_scale"), (dict(workspace_bytes=48 + 639), "workspace"), (dict(x=P + 1), "aligned"),
    (dict(y=P), "overlap"),
])
def test_exact_matmul_refuses(moe, bad, msg):
    _refused("moe_fp8_matmul_exact_async", {**MM, **bad}, msg)


def test_no_rows_are_no_work(moe):
    from mixtureofexperts_amd import _lib

    assert _lib.lib().moe_fp8_matmul_exact_async(*{**MM, "rows": 0, "workspace": None, "x": None}.values()) == 0
