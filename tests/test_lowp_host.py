"""Refusals of the low-precision and grouped products, all before any device call (CPU)."""
import ctypes

import numpy as np
import pytest


@pytest.fixture()
def buf():
    return (ctypes.c_char * 4096)()


def refused(lib, name, *args):
    assert getattr(lib, name)(*args) != 0
    return lib.cudeep_b200_last_error().decode()


def test_c_abi_refusals(lib, buf):
    p = ctypes.addressof(buf)
    p += -p % 16
    assert "null" in refused(lib, "cudeep_b200_quantize_fp8", None, 0, 4, 128, 1, p, p, None)
    assert "type" in refused(lib, "cudeep_b200_quantize_fp8", p, 3, 4, 128, 1, p, p, None)
    assert "1 or 128 rows" in refused(lib, "cudeep_b200_quantize_fp8", p, 0, 4, 128, 64, p, p, None)
    assert "negative" in refused(lib, "cudeep_b200_quantize_fp8", p, 0, -1, 128, 1, p, p, None)
    assert "positive" in refused(lib, "cudeep_b200_quantize_fp8", p, 0, 4, 0, 1, p, p, None)
    assert "aligned" in refused(lib, "cudeep_b200_quantize_fp8", p + 1, 2, 4, 128, 1, p, p, None)
    assert "aligned" in refused(lib, "cudeep_b200_quantize_fp8", p, 2, 4, 128, 1, p, p + 2, None)
    assert "null" in refused(lib, "cudeep_b200_dequantize_fp8", p, None, 4, 128, 1, p, 0, None)
    assert "type" in refused(lib, "cudeep_b200_cast", p, 0, p, 7, 4, None)
    for name in ("cudeep_b200_grouped_matmul_nt", "cudeep_b200_grouped_matmul_nn"):
        assert "null" in refused(lib, name, p, p, p, 2, None, 4, 8, 8, 8, None)
        assert "16-bit" in refused(lib, name, p, p, p, 0, p, 4, 8, 8, 8, None)
        assert "groups" in refused(lib, name, p, p, p, 2, p, 0, 8, 8, 8, None)
        assert "groups" in refused(lib, name, p, p, p, 2, p, 1025, 8, 8, 8, None)
        assert "negative" in refused(lib, name, p, p, p, 2, p, 4, -8, 8, 8, None)
        assert "positive" in refused(lib, name, p, p, p, 2, p, 4, 8, 8, 0, None)
        assert "aligned" in refused(lib, name, p, p + 1, p, 2, p, 4, 8, 8, 8, None)
    assert "operands' type" in refused(lib, "cudeep_b200_grouped_matmul_tn", p, p, p, 2, 1, p, 4, 8, 8, 8, None)
    assert "epilogue" in refused(lib, "cudeep_b200_linear_forward_fp8", p, p, p, p, None, p, 0, 4, 4, 4, 9, None)
    assert "null" in refused(lib, "cudeep_b200_linear_forward_fp8", p, None, p, p, None, p, 0, 4, 4, 4, 0, None)
    assert "positive" in refused(lib, "cudeep_b200_linear_forward_fp8", p, p, p, p, None, p, 0, 4, 0, 4, 0, None)
    assert "null" in refused(lib, "cudeep_b200_linear_backward_data_fp8", p, p, p, p, None, 0, 4, 4, 4, None)
    saved = "cudeep_b200_linear_backward_saved_fp8"
    assert "no gradient" in refused(lib, saved, p, 2, p, p, p, p, 0, p, None, None, 2, None, 4, 4, 4, None)
    assert "needs W" in refused(lib, saved, p, 2, p, p, p, p, 0, None, p, p, 2, p, 4, 4, 4, None)
    assert "needs x8" in refused(lib, saved, p, 2, None, p, p, p, 0, p, p, p, 2, p, 4, 4, 4, None)
    assert "needs z8" in refused(lib, saved, p, 2, p, p, None, p, 2, p, p, p, 2, p, 4, 4, 4, None)
    assert "of dy's type" in refused(lib, saved, p, 2, p, p, p, p, 0, p, p, p, 1, p, 4, 4, 4, None)
    assert "16-bit" in refused(lib, saved, p, 0, p, p, p, p, 0, p, p, p, 0, p, 4, 4, 4, None)


def test_no_rows_needs_no_device(lib, buf):
    """Products of no rows are done before any device call (those that write nothing)."""
    p = ctypes.addressof(buf)
    p += -p % 16
    assert lib.cudeep_b200_quantize_fp8(p, 0, 0, 128, 1, p, p, None) == 0
    assert lib.cudeep_b200_linear_forward_fp8(p, p, p, p, None, p, 0, 0, 4, 4, 0, None) == 0
    assert lib.cudeep_b200_linear_backward_data_fp8(p, p, p, p, p, 0, 0, 4, 4, None) == 0
    assert lib.cudeep_b200_grouped_matmul_nt(p, p, p, 2, p, 4, 0, 8, 8, None) == 0
    assert lib.cudeep_b200_grouped_matmul_nn(p, p, p, 2, p, 4, 0, 8, 8, None) == 0
    assert lib.cudeep_b200_cast(p, 0, p, 2, 0, None) == 0


@pytest.fixture()
def cd(monkeypatch):
    import cudeep_b200
    from cudeep_b200 import tensor

    class FakeStorage:
        def __init__(self, nbytes):
            self.ptr = None
            self.nbytes = nbytes

    monkeypatch.setattr(tensor, "_Storage", FakeStorage)
    return cudeep_b200


def test_low_precision_tensors(cd):
    D = cd.DType
    assert cd.Tensor([3, 5], D.bfloat16).nbytes() == 30
    assert cd.Tensor([3, 5], D.float8_e4m3).nbytes() == 15
    assert cd.Tensor([4], D.int32).nbytes() == 16
    with pytest.raises(RuntimeError):
        cd.Tensor([2], D.float16)
    b = cd.Tensor([4, 4], D.bfloat16)
    for call in (lambda: b.matmul(b), lambda: b.fill_(1.0), lambda: cd.linear(b, b), lambda: cd.broadcast_add(b, cd.Tensor([4], D.bfloat16)),
                 lambda: b.relu(), lambda: b.transpose(0, 1).contiguous(), lambda: cd.Tensor.randn([2], D.int32),
                 lambda: cd.Tensor([4], D.int32).to(D.float32),
                 lambda: cd.conv2d(cd.Tensor([1, 3, 8, 8], D.bfloat16), cd.Tensor([4, 3, 3, 3], D.bfloat16))):
        with pytest.raises(RuntimeError):
            call()


def test_e4m3_values():
    from cudeep_b200.tensor import _e4m3_values
    v = _e4m3_values()
    assert v[0x7e] == 448 and v[1] == 2.0 ** -9 and v[0x38] == 1 and v[0xb8] == -1 and np.isnan(v[[0x7f, 0xff]]).all()
    torch = pytest.importorskip("torch")
    want = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(v, want, equal_nan=True)


def test_python_refusals(cd):
    D = cd.DType
    T = cd.Tensor

    def rows8(r, c):
        return cd.Fp8Tensor(T([r, c], D.float8_e4m3), T([-(-c // 128), r]), False)

    def tiles8(r, c):
        return cd.Fp8Tensor(T([r, c], D.float8_e4m3), T([-(-r // 128), -(-c // 128)]), True)

    with pytest.raises(RuntimeError, match="match the matrix"):
        cd.Fp8Tensor(T([4, 300], D.float8_e4m3), T([2, 4]), False)
    with pytest.raises(RuntimeError, match="float8_e4m3 expected"):
        cd.Fp8Tensor(T([4, 300]), T([3, 4]), False)
    with pytest.raises(RuntimeError, match="2-D"):
        cd.quantize_fp8(T([4]))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        cd.quantize_fp8(T([4, 4], D.float64))
    with pytest.raises(RuntimeError, match="contiguous"):
        cd.quantize_fp8(T([4, 8]).transpose(0, 1))
    with pytest.raises(RuntimeError, match="1 x 128"):
        cd.linear_fp8(tiles8(4, 8), tiles8(8, 8))
    with pytest.raises(RuntimeError, match="tiles=True"):
        cd.linear_fp8(rows8(4, 8), rows8(8, 8))
    with pytest.raises(RuntimeError, match="inner"):
        cd.linear_fp8(rows8(4, 8), tiles8(8, 16))
    with pytest.raises(RuntimeError, match="out_features"):
        cd.linear_fp8(rows8(4, 8), tiles8(6, 8), T([5]))
    with pytest.raises(RuntimeError, match="unknown activation"):
        cd.linear_fp8(rows8(4, 8), tiles8(6, 8), None, "tanh")
    with pytest.raises(RuntimeError, match="inner"):
        cd.linear_fp8_backward_data(rows8(4, 8), tiles8(6, 8))
    b = lambda *s: T(list(s), D.bfloat16)      # noqa: E731
    with pytest.raises(RuntimeError, match="needs z"):
        cd.linear_backward_saved(b(4, 6), rows8(4, 8), b(6, 8), None, "gelu")
    with pytest.raises(RuntimeError, match="x \\[m, k\\]"):
        cd.linear_backward_saved(b(4, 6), rows8(5, 8), b(6, 8))
    with pytest.raises(RuntimeError, match="one element more"):
        cd.grouped_linear(b(4, 8), b(3, 6, 8), T([3], D.int32))
    with pytest.raises(RuntimeError, match="int32"):
        cd.grouped_linear(b(4, 8), b(2, 6, 8), T([3]))
    with pytest.raises(RuntimeError, match="inner"):
        cd.grouped_linear(b(4, 9), b(2, 6, 8), T([3], D.int32))
    with pytest.raises(RuntimeError, match="grad"):
        cd.grouped_linear_backward(b(4, 7), b(4, 8), b(2, 6, 8), T([3], D.int32))


HUGE = 2147483647


@pytest.mark.parametrize("m,n,k", [(HUGE, 8, 8), (8, HUGE, 8), (8, 8, HUGE), (HUGE - 65535 + 1, 8, 8)])
def test_extents_near_the_end_of_32_bits_are_refused(lib, buf, m, n, k):
    """Beyond 2^31 - 65536 the kernels' and planners' sums of an extent and a tile would wrap around."""
    p = ctypes.addressof(buf)
    p += -p % 16
    assert "at most" in refused(lib, "cudeep_b200_linear_forward_fp8", p, p, p, p, None, p, 0, m, n, k, 0, None)
    assert "at most" in refused(lib, "cudeep_b200_linear_backward_data_fp8", p, p, p, p, p, 0, m, n, k, None)
    assert "at most" in refused(lib, "cudeep_b200_linear_backward_saved_fp8", p, 2, p, p, p, p, 2, p, p, p, 2, p, m, n, k, None)
    for name in ("cudeep_b200_grouped_matmul_nt", "cudeep_b200_grouped_matmul_nn"):
        assert "at most" in refused(lib, name, p, p, p, 2, p, 4, m, n, k, None)
    assert "at most" in refused(lib, "cudeep_b200_grouped_matmul_tn", p, p, p, 2, 0, p, 4, m, n, k, None)
    if k != 8:
        assert "at most" in refused(lib, "cudeep_b200_quantize_fp8", p, 2, 1, k, 1, p, p, None)
        assert "at most" in refused(lib, "cudeep_b200_dequantize_fp8", p, p, 1, k, 1, p, 2, None)


def test_rows_of_more_bytes_than_a_copy_counts_are_refused(lib, buf):
    """Rows that are no 16-byte multiples are copied, counted in bytes by 32 bits.  (Aligned ones of that length are not copied.)"""
    p = ctypes.addressof(buf)
    p += -p % 16
    long = (1 << 30) + 1
    for name in ("cudeep_b200_grouped_matmul_nt", "cudeep_b200_grouped_matmul_nn"):
        assert "row" in refused(lib, name, p, p, p, 2, p, 4, 4, 8, long, None)
    assert "row" in refused(lib, "cudeep_b200_grouped_matmul_tn", p, p, p, 2, 0, p, 4, 4, 8, long, None)
    assert "row" in refused(lib, "cudeep_b200_linear_backward_saved_fp8", p, 2, p, p, p, p, 2, p, p, p, 2, p, 4, 8, long, None)
    assert "2^29" in refused(lib, "cudeep_b200_linear_backward_saved_fp8", p, 1, p, p, p, p, 2, p, p, p, 1, p, (1 << 29) + 1, 8, 8,
                             None)
