"""Blocks of 8-bit floating point (e4m3 with a power-of-two scale for each 128 columns) against a restatement in 64 bits.

Nothing here has a tolerance: a scale is a power of two found exactly, the division by it is exact, and the one rounding to
e4m3 is to nearest even, so bytes and scales have to be equal.
"""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "f16": 1, "bf16": 2}


def e4m3_table(torch):
    """The 127 non-negative values of e4m3 in code order."""
    codes = torch.arange(127, dtype=torch.float64)
    e, m = torch.div(codes, 8, rounding_mode="floor"), codes % 8
    return torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e - 7))


def round_e4m3(torch, v):
    """Codes of v (float64, |v| <= 448) rounded to nearest, ties to the even code."""
    table = e4m3_table(torch).to(v.device)
    a = v.abs()
    hi = torch.searchsorted(table, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - table[lo], table[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(table[hi] == a, hi, code)
    return code + 128 * torch.signbit(v)


def reference(torch, x, block_rows):
    rows, cols = x.shape
    wide = x.double()
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    p = torch.zeros(rb * block_rows, cb * 128, dtype=torch.float64, device=x.device)
    p[:rows, :cols] = torch.where(torch.isfinite(wide), wide, torch.zeros_like(wide)).abs()
    amax = p.view(rb, block_rows, cb, 128).amax(dim=(1, 3))
    scale = torch.exp2(torch.floor(torch.log2(amax / 448)) - 1)
    for _ in range(3):
        scale = torch.where(amax / scale > 448, scale * 2, scale)
    scale = torch.where(amax == 0, torch.ones_like(scale), scale.clamp(min=2.0 ** -126))
    spread = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    finite = torch.isfinite(wide)
    code = round_e4m3(torch, torch.where(finite, wide, torch.zeros_like(wide)) / spread)
    code = torch.where(finite, code, torch.full_like(code, 127)).to(torch.uint8)
    return code, (scale.t() if block_rows == 1 else scale).float().contiguous()


def quantize(dev, x, block_rows, stream=None):
    torch = dev.torch
    rows, cols = x.shape
    q = torch.full((rows, cols), 0xAA, dtype=torch.uint8, device=dev.dev)
    cb = -(-cols // 128)
    scales = dev.empty((cb, rows) if block_rows == 1 else (-(-rows // 128), cb))
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
    dev.check(dev.lib.cudeep_b200_quantize_fp8(dev.ptr(x), code, rows, cols, block_rows, dev.ptr(q), dev.ptr(scales),
                                               stream))
    return q, scales


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 129), (33, 1000), (128, 256), (130, 515), (257, 2048)])
def test_quantize_is_exact(dev, shape, dtype, block_rows):
    torch = dev.torch
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    gen = torch.Generator(device=dev.dev).manual_seed(shape[0] * 1000 + shape[1])
    x = torch.randn(shape, generator=gen, device=dev.dev) * torch.exp(
        2 * torch.randn(shape[0], 1, generator=gen, device=dev.dev))
    x = x.to(t)
    q, scales = quantize(dev, x, block_rows)
    want_q, want_s = reference(torch, x, block_rows)
    assert torch.equal(scales, want_s)
    assert torch.equal(q, want_q)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_borders(dev, block_rows):
    """Ties, the largest finite value's neighbourhood, subnormals, zeros, infinities and NaN."""
    torch = dev.torch
    x = torch.zeros(140, 300, device=dev.dev)
    x[0, :6] = torch.tensor([448.0, 232.0, 17.0, 19.0, 2.0 ** -9, 2.0 ** -10])       # ties between codes at scale 1
    x[1, :3] = torch.tensor([448.00003, 447.99997, -448.00003])                       # just above: the next scale
    x[2, 0] = 1e-45                                                                   # the smallest subnormal
    x[3, 0] = 3.4028234e38
    x[4, 5:8] = torch.tensor([float("inf"), -float("inf"), float("nan")])
    x[4, 8] = 3.0
    x[130, 290] = float("nan")                                                        # a block with nothing finite but zeros
    x[131, 0] = -0.0
    q, scales = quantize(dev, x, block_rows)
    want_q, want_s = reference(torch, x, block_rows)
    assert torch.equal(scales, want_s)
    assert torch.equal(q, want_q)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("lead,shift", [(0, 0), (0, 1), (4, 0), (8, 4), (3, 2)])
def test_quantize_odd_rows_at_any_address(dev, block_rows, lead, shift):
    """Rows whose starts take all phases within a word, from bases that suit vectors and from others."""
    torch = dev.torch
    rows, cols = 131, 389
    for t in (torch.float32, torch.bfloat16):
        buf = torch.randn(rows * cols + lead, device=dev.dev).to(t)
        x = buf[lead:].view(rows, cols)
        out = torch.full((rows * cols + 64,), 0xAA, dtype=torch.uint8, device=dev.dev)
        scales = dev.empty((4, rows) if block_rows == 1 else (2, 4))
        dev.check(dev.lib.cudeep_b200_quantize_fp8(dev.ptr(x), 0 if t == torch.float32 else 2, rows, cols, block_rows,
                                                   ctypes.c_void_p(out.data_ptr() + 16 + shift), dev.ptr(scales), None))
        want_q, want_s = reference(torch, x, block_rows)
        start, end = 16 + shift, 16 + shift + rows * cols
        assert torch.equal(out[start:end].view(rows, cols), want_q) and torch.equal(scales, want_s)
        assert bool((out[:start] == 0xAA).all()) and bool((out[end:] == 0xAA).all())


def test_quantize_unaligned_base_and_neighbours(dev):
    """A matrix that starts one element into a buffer; bytes around the result stay as they were."""
    torch = dev.torch
    rows, cols = 37, 264
    buf = torch.randn(rows * cols + 1, device=dev.dev).to(torch.bfloat16)
    x = buf[1:].view(rows, cols)
    out = torch.full((rows * cols + 32,), 0xAA, dtype=torch.uint8, device=dev.dev)
    scales = dev.empty((3, rows))
    dev.check(dev.lib.cudeep_b200_quantize_fp8(dev.ptr(x), 2, rows, cols, 1, ctypes.c_void_p(out.data_ptr() + 16),
                                               dev.ptr(scales), None))
    want_q, want_s = reference(torch, x, 1)
    assert torch.equal(out[16:-16].view(rows, cols), want_q) and torch.equal(scales, want_s)
    assert bool((out[:16] == 0xAA).all()) and bool((out[-16:] == 0xAA).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_dequantize_every_code(dev, block_rows, dtype):
    """All 256 codes under several scales: one rounding to the result's type, which torch's conversion makes too."""
    torch = dev.torch
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    q = torch.arange(256, dtype=torch.int32, device=dev.dev).to(torch.uint8).repeat(130, 1)
    scales = torch.exp2(torch.randint(-20, 12, (2, 130) if block_rows == 1 else (2, 2), device=dev.dev).float())
    y = dev.empty((130, 256), dtype=t)
    dev.check(dev.lib.cudeep_b200_dequantize_fp8(dev.ptr(q), dev.ptr(scales), 130, 256, block_rows, dev.ptr(y),
                                                 CODES[dtype], None))
    spread = (scales.t().repeat_interleave(128, 1) if block_rows == 1
              else scales.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1))
    want = (q.view(torch.float8_e4m3fn).double() * spread.double()).to(t)
    assert torch.equal(torch.nan_to_num(y, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert torch.equal(y.isnan(), want.isnan())


def test_no_rows(dev):
    torch = dev.torch
    x = torch.empty(0, 128, device=dev.dev)
    one = torch.empty(1, device=dev.dev)
    dev.check(dev.lib.cudeep_b200_quantize_fp8(dev.ptr(one), 0, 0, 128, 1, dev.ptr(one), dev.ptr(one), None))
    dev.check(dev.lib.cudeep_b200_dequantize_fp8(dev.ptr(one), dev.ptr(one), 0, 128, 1, dev.ptr(one), 0, None))
    assert x.numel() == 0 and dev.sync_status() == 0
