"""8-bit Linear products and the backward pass from 8-bit activations against the same formulas in 64 bits.

Tolerances.  Products of e4m3 values (four significant bits each) are exact in FP32.  A block of 128 of them is summed by
the tensor core, which may truncate each partial sum (128 * 2^-23 of the block's sum of magnitudes), and the scaled blocks
are added in FP32 with one fused multiply-add each (2^-24 of the running sum, once per block, and one rounding of the
product of the scales, exact for powers of two): together (128 + blocks) * 2^-23 of the sum of magnitudes.  A 16-bit result
adds torch.finfo(t).eps / 2 of its value.  The epilogue's activations have slopes of at most 1.13 and are computed with
approximate ex2 and rcp (2 ulp each, on terms of the size of the result or of 1): 2^-20 of max(1, |z|) covers them.
"""
import pytest

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def random_fp8(dev, rows, cols, block_rows, gen, pow2=True):
    """Codes without NaN, and scales; and the values they stand for in 64 bits."""
    torch = dev.torch
    q = torch.randint(0, 256, (rows, cols), generator=gen, device=dev.dev, dtype=torch.int32)
    q = torch.where(q % 128 == 127, q - 1, q).to(torch.uint8)
    cb, rb = -(-cols // 128), -(-rows // block_rows)
    shape = (cb, rows) if block_rows == 1 else (rb, cb)
    if pow2:
        scales = torch.exp2(torch.randint(-9, -4, shape, generator=gen, device=dev.dev).float())
    else:
        scales = torch.rand(shape, generator=gen, device=dev.dev) * 0.02 + 0.001
    spread = (scales.t() if block_rows == 1 else scales.repeat_interleave(128, 0)[:rows]).repeat_interleave(128, 1)[:, :cols]
    return q, scales, q.view(torch.float8_e4m3fn).double() * spread.double()


def act64(torch, z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    return z


def check(torch, got, want, bound):
    info = torch.finfo(got.dtype)
    if got.dtype != torch.float32:
        bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps
    assert not got.isnan().any()
    worst = ((got.double() - want).abs() - bound).max().item()
    assert worst <= 0, worst


SHAPES = [(1, 64, 64), (3, 128, 128), (16, 256, 384), (33, 130, 300), (100, 77, 1001), (129, 520, 128), (257, 256, 256),
          (300, 1000, 520), (512, 384, 2048), (16, 256, 4096), (7, 4200, 4200), (128, 300, 2000), (809, 104, 3000), (1119, 117, 536)]


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(dev, m, n, k, out):
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(m * 7 + n)
    x8, xs, x = random_fp8(dev, m, k, 1, gen)
    w8, ws, w = random_fp8(dev, n, k, 128, gen)
    y = torch.full((m, n), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), None, dev.ptr(y),
                                                     CODES[out], m, n, k, 0, None))
    assert dev.sync_status() == 0
    check(torch, y, x @ w.t(), (128 + -(-k // 128)) * 2.0 ** -23 * (x.abs() @ w.abs().t()))


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("pow2", [True, False])
def test_forward_bias_activation_and_any_scales(dev, act, pow2):
    torch = dev.torch
    m, n, k = 70, 200, 400
    gen = torch.Generator(device=dev.dev).manual_seed(5)
    x8, xs, x = random_fp8(dev, m, k, 1, gen, pow2)
    w8, ws, w = random_fp8(dev, n, k, 128, gen, pow2)
    bias = torch.randn(n, generator=gen, device=dev.dev)
    ws = ws * 2.0 ** -8      # pre-activations of a few units
    w = w * 2.0 ** -8
    y = torch.full((m, n), float("nan"), device=dev.dev)
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), dev.ptr(bias),
                                                     dev.ptr(y), 0, m, n, k, ACTS[act], None))
    assert dev.sync_status() == 0
    z = x @ w.t() + bias.double()
    bound = (128 + 4 + 1) * 2.0 ** -23 * (x.abs() @ w.abs().t() + bias.double().abs())
    if act != "none":
        bound = 1.13 * bound + 2.0 ** -20 * z.abs().clamp(min=1)
    check(torch, y, act64(torch, z, act), bound)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward_data(dev, m, n, k, out):
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(m * 11 + k)
    d8, ds, dy = random_fp8(dev, m, n, 1, gen)
    w8, ws, w = random_fp8(dev, n, k, 128, gen)
    dx = torch.full((m, k), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    dev.check(dev.lib.cudeep_b200_linear_backward_data_fp8(dev.ptr(d8), dev.ptr(ds), dev.ptr(w8), dev.ptr(ws), dev.ptr(dx),
                                                           CODES[out], m, n, k, None))
    assert dev.sync_status() == 0
    check(torch, dx, dy @ w, (128 + -(-n // 128)) * 2.0 ** -23 * (dy.abs() @ w.abs()))


@pytest.mark.parametrize("scales", ["pow2", "any", "one_odd"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(4096, 4096, 4096), (2900, 5003, 4200), (6000, 2560, 6500)])
def test_large_products(dev, m, n, k, out, scales):
    """Sizes at which the tensor core applies the scales if all are powers of two, and does not if one is none.  There its sums
    run over up to 2048 (FP32) or 16384 elements of K, 32 to a step, each step truncated."""
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(m + k)
    t = dtype_of(torch, out)
    x8, xs, x = random_fp8(dev, m, k, 1, gen, scales != "any")
    w8, ws, w = random_fp8(dev, n, k, 128, gen, scales != "any")
    if scales == "one_odd":
        xs[-1, -1] = 0.3
        x[-1, (k - 1) // 128 * 128:] = (x8[-1, (k - 1) // 128 * 128:].view(torch.float8_e4m3fn).double() * xs[-1, -1].double())
    y = torch.full((m, n), float("nan"), device=dev.dev, dtype=t)
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), None, dev.ptr(y),
                                                     CODES[out], m, n, k, 0, None))
    assert dev.sync_status() == 0
    check(torch, y, x @ w.t(), (128 + -(-k // 128)) * 2.0 ** -23 * (x.abs() @ w.abs().t()))
    if k % 128 or n % 128:
        return
    dx = torch.full((m, k), float("nan"), device=dev.dev, dtype=t)
    dev.check(dev.lib.cudeep_b200_linear_backward_data_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), dev.ptr(dx),
                                                           CODES[out], m, k, n, None))
    assert dev.sync_status() == 0
    check(torch, dx, x @ w, (128 + -(-k // 128)) * 2.0 ** -23 * (x.abs() @ w.abs()))


def slope64(torch, z, name):
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(act64(torch, z, name).sum(), z)[0] if name != "none" else torch.ones_like(z)


@pytest.mark.parametrize("dw_type", ["same", "f32"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (40, 130, 72), (333, 77, 101), (300, 256, 384), (2500, 64, 136), (1100, 512, 512),
                                   (150, 2600, 1900)])
def test_backward_saved(dev, m, n, k, act, dtype, dw_type):
    """dz is rounded to the type first (eps / 2 of it): that much of the sum of magnitudes joins the products' bounds."""
    torch = dev.torch
    t = dtype_of(torch, dtype)
    gen = torch.Generator(device=dev.dev).manual_seed(m + n + k)
    x8, xs, x = random_fp8(dev, m, k, 1, gen)
    z8, zs, z = random_fp8(dev, m, n, 1, gen)
    w = (torch.randn(n, k, generator=gen, device=dev.dev) / n ** 0.5).to(t)
    dy = torch.randn(m, n, generator=gen, device=dev.dev).to(t)
    to = torch.float32 if dw_type == "f32" else t
    dx = torch.full((m, k), float("nan"), device=dev.dev, dtype=t)
    dw = torch.full((n, k), float("nan"), device=dev.dev, dtype=to)
    db = torch.full((n,), float("nan"), device=dev.dev)
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(
        dev.ptr(dy), CODES[dtype], dev.ptr(x8), dev.ptr(xs), dev.ptr(z8), dev.ptr(zs), ACTS[act], dev.ptr(w), dev.ptr(dx),
        dev.ptr(dw), 0 if dw_type == "f32" else CODES[dtype], dev.ptr(db), m, n, k, None))
    assert dev.sync_status() == 0
    slope = slope64(torch, z, act)
    dz = dy.double() * slope
    # The slope in FP32: terms of at most 1.13 and, for GELU and SiLU, z times a factor below 1: 2^-20 of max(1, |z|) in all.
    off = dy.double().abs() * (2.0 ** -20 * z.abs().clamp(min=1) if act != "none" else 0 * z)
    half = torch.finfo(t).eps / 2
    rounded = off + (half * dz.abs() + torch.finfo(t).smallest_normal * half if act != "none" else 0 * dz)
    w64 = w.double()
    check(torch, db, dz.sum(0), off.sum(0) + m * 2.0 ** -24 * dz.abs().sum(0))
    check(torch, dx, dz @ w64, rounded @ w64.abs() + n * 2.0 ** -23 * (dz.abs() @ w64.abs()))
    # FP16: x relative to its block's largest scale is off by at most 2^-25 of that scale (half a subnormal step).
    lost = 0 * x
    if dtype == "f16":
        lost = (xs.amax(1).double() * 2.0 ** -25).repeat_interleave(128)[None, :k].expand(m, k)
    check(torch, dw, dz.t() @ x, rounded.t() @ x.abs() + dz.abs().t() @ lost + m * 2.0 ** -23 * (dz.abs().t() @ x.abs()))


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k", [(4, 256, 256), (4, 300, 4096), (1100, 4096, 512), (300, 520, 256), (4096, 4096, 2048)])
def test_activations_of_infinities_huge_values_and_nan(dev, act, m, n, k):
    """Features of one sign each, so that a row's pre-activation is +-s: infinite, huge, NaN or moderate by the row.

    Below z = -64 the activated values are within 2^-54 of their limit 0 (sigmoid: 2^-60); everything here is a sum of equal
    terms that are powers of two times 448, whose FP32 sums lose at most the tolerance of the other tests."""
    torch = dev.torch
    x8 = torch.full((m, k), 0x38, device=dev.dev, dtype=torch.uint8)      # 1.0
    w8 = torch.full((n, k), 0x7E, device=dev.dev, dtype=torch.uint8)      # 448
    w8[1::2] = 0xFE
    xs = torch.full((-(-k // 128), m), 2.0 ** -36, device=dev.dev)
    xs[:, 0] = 2.0 ** 100
    xs[:, 1] = 2.0 ** 80
    x8[2, k // 2] = 0x7F      # NaN
    ws = torch.full((-(-n // 128), -(-k // 128)), 2.0 ** 20, device=dev.dev)
    y = torch.zeros((m, n), device=dev.dev)
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), None, dev.ptr(y), 0,
                                                     m, n, k, ACTS[act], None))
    assert dev.sync_status() == 0
    up, down = y[:, 0::2], y[:, 1::2]
    inf = float("inf")
    if act == "relu":      # drops NaN, as the framework's other epilogues
        assert (y[2] == 0).all() and not y.isnan().any()
    else:
        assert y[2].isnan().all() and y.isnan().sum().item() == n
    if act == "sigmoid":
        assert (up[:2] == 1).all()
    else:
        assert (up[0] == inf).all()
        assert ((up[1].double() / (448.0 * k * 2.0 ** 100) - 1).abs() <= (128 + k // 128) * 2.0 ** -23 + 2.0 ** -20).all()
    if act == "none":
        assert (down[0] == -inf).all() and (down[1] == -up[1, :1]).all()
    else:
        assert (down[:2].abs() <= 2.0 ** -54).all()
    z = 448.0 * k * 2.0 ** -16 * torch.ones(n, device=dev.dev, dtype=torch.float64)
    bound = 1.13 * (128 + k // 128) * 2.0 ** -23 * z + 2.0 ** -20 * z.clamp(min=1)
    z[1::2] *= -1
    check(torch, y[3:], act64(torch, z, act).expand(m - 3, n), bound)
