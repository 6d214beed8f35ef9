"""Which kernel a product takes: the tests of its forms (test_gpu_ops_grouped.py,
test_gpu_ops_int8.py) claim tile sizes, split sums and the streamed form at most of
the sizes below."""
import re
import warnings

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FLUX, LLAMA = 0, 1
F32, BF16, I8 = 0, 1, 2
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _kernels(call):
    """{kernel name: template arguments} of the operators' kernels that call() launches."""
    from torch.profiler import ProfilerActivity, profile

    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
    got = {}
    for e in p.key_averages():
        m = re.search(r"moe::ops::(\w+)(?:<([^>]*)>)?\(", e.key)
        if m:
            got[m.group(1)] = [v.strip() for v in (m.group(2) or "").split(",")]
    return got


def _operands(lens, K, N, dtype, layout):
    off = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    M, E = sum(lens), len(lens)
    z = lambda *s: torch.zeros(*s, dtype=DT[dtype], device="cuda")
    return z(M, K), z(M, N), z(E, *((N, K) if layout == LLAMA else (K, N))), off


def _tile(got):
    """(rows, columns) of op_gemm_kernel's tiles and the alignment of its loads."""
    a = got["op_gemm_kernel"]
    return (int(a[4]), int(a[5])), int(a[11])


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_rows_products(moe, layout):
    col = layout == FLUX  # the forward product's weights are strided along k
    for lens, K, N, dtype, tile, split in (
        ([2100, 1, 3000, 3400], 136, 4040, "bf16", 256, False),
        ([700, 0, 900, 500], 72, 2048, "bf16", 128, False),
        ([33, 130, 5, 0, 300], 200, 136, "bf16", 64, False),
        ([71], 5440, 64, "bf16", 64, True),
        ([71], 5440, 64, "f32", 64, True),
        ([1], 8192, 16, "f32", 64 if col else 0, True),
        ([3, 0, 2], 16401, 125, "f32", 64 if col else 0, True),
        ([3, 0, 2], 64, 96, "bf16", 64 if col else 0, False),
        ([3, 0, 2], 64, 8200, "bf16", 64, False),
        ([3, 0, 2], 64, 96, "f32", 64 if col else 0, False),
        ([8, 3, 13], 2048, 96, "bf16", 64 if col else 0, True if col else False),
        ([8, 3, 14], 2048, 96, "bf16", 64, True),
        ([3000], 96, 3000, "f32", 64, False),
        ([2048], 96, 4096, "f32", 128, False),
        ([17, 0, 1, 64], 64, 96, "f32", 64, False),
    ):
        x, dy, w, off = _operands(lens, K, N, dtype, layout)
        got = _kernels(lambda: moe.grouped_matmul(x, w, off, layout=layout))
        print("forward", lens, K, N, dtype, got, flush=True)
        assert ("op_fold_kernel" in got) == split
        if tile == 0:
            assert "op_stream_kernel" in got and "op_gemm_kernel" not in got
        else:
            assert "op_stream_kernel" not in got and _tile(got)[0] == (tile, tile)
    # the row gradient reads the weights along their other side
    x, dy, w, off = _operands([2100, 1, 3000, 3400], 4040, 136, "bf16", layout)
    got = _kernels(lambda: moe.grouped_matmul_grad_x(dy, w, off, layout=layout))
    assert _tile(got) == ((256, 256), 16) and got["op_gemm_kernel"][2] == ("false" if col else "true")


@pytest.mark.parametrize("layout", [LLAMA, FLUX])
def test_weight_gradients(moe, layout):
    for lens, K, N, dtype, tile, split in (
        ([70, 0, 133], 4096, 2040, "bf16", 128, False),  # one and a half rounds of 256 x 256
        ([70, 0, 133, 9], 4096, 2040, "bf16", 256, False),
        ([70, 0, 64, 1, 200, 66, 2, 30], 2048, 2040, "bf16", 256, False),
        ([100, 40, 0, 64], 1024, 1024, "bf16", 128, False),
        ([100, 40, 0, 64], 1024, 1024, "f32", 128, False),
        ([33, 130, 5, 0, 300], 200, 136, "bf16", 64, False),
        ([3000], 96, 40, "bf16", 64, True),
        ([2500, 0, 4000], 64, 64, "f32", 64, True),
        ([4000], 2048, 640, "f32", 64, True),
        ([4096], 1024, 1024, "f32", 64, True),
        ([300, 900], 2048, 2048, "f32", 128, False),
    ):
        x, dy, w, off = _operands(lens, K, N, dtype, layout)
        got = _kernels(lambda: moe.grouped_matmul_grad_w(x, dy, off, layout=layout, out_dtype=torch.float32))
        print("weight gradient", lens, K, N, dtype, got, flush=True)
        assert _tile(got)[0] == (tile, tile) and ("op_fold_kernel" in got) == split


def test_loads_by_alignment(moe):
    # 16: aligned rows; 4: rows of whole dwords; 0: through registers
    for K, N, dtype, vb in ((200, 136, "bf16", 16), (202, 134, "bf16", 4), (201, 135, "bf16", 0), (201, 135, "f32", 4)):
        x, dy, w, off = _operands([33, 130, 5, 0, 300], K, N, dtype, LLAMA)
        for call in (lambda: moe.grouped_matmul(x, w, off), lambda: moe.grouped_matmul_grad_x(dy, w, off),
                     lambda: moe.grouped_matmul_grad_w(x, dy, off)):
            assert _tile(_kernels(call))[1] == vb, (K, N, dtype)


def test_int8_products(moe):
    for lens, K, N, tile, split in (([3000, 5500], 160, 4112, 256, False), ([700, 0, 900, 500], 144, 2048, 128, False),
                                    ([33, 130, 5, 0, 300], 208, 136, 64, False), ([40, 30], 20000, 33, 64, True),
                                    ([0, 3, 0], 7, 5, 0, False), ([0, 9, 0], 4096, 8200, 0, False), ([0, 9, 0], 2048, 8200, 64, False),
                                    ([0, 9, 0], 5001, 50, 64, True), ([0, 0, 2, 0, 1, 0, 0], 20000, 17, 0, True)):
        x, _, w, off = _operands(lens, K, N, "bf16", LLAMA)
        ws = torch.ones(w.shape[:2], device="cuda")
        w = w.to(torch.int8)
        got = _kernels(lambda: moe.int8_matmul(x, w, ws, off))
        print("int8", lens, K, N, got, flush=True)
        assert any(n.startswith("quantize_i8") for n in got) and ("op_fold_kernel" in got) == split
        if tile == 0:
            assert "op_stream_kernel" in got and "op_gemm_kernel" not in got
        else:
            assert _tile(got)[0] == (tile, tile)
