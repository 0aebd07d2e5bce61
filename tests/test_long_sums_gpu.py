"""Sums over many rows or columns.  All terms are positive, so that what a truncating accumulator drops adds up."""
import pytest

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "f16": 1, "bf16": 2}
HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def positive(dev, rows, cols, t, gen, scale):
    torch = dev.torch
    return ((torch.rand(rows, cols, generator=gen, device=dev.dev) + 1) * scale).to(t)


def product64(torch, a, b):
    """a^T b in 64 bits, a range of rows at a time."""
    return sum(x.double().t() @ y.double() for x, y in zip(a.split(1 << 16), b.split(1 << 16)))


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,n,k", [(1_000_003, 64, 72), (200_001, 640, 512), (16385, 136, 264)])
def test_gradient_over_many_rows(dev, rows, n, k, dtype, out, grouped):
    """At most 16384 rows (FP32 result: 2048) go through the tensor core's accumulator at once; however it orders them, each drops
    at most 2^-23 of the sum so far: 2^-9 (2^-12) of the result.  Adding up such sums in FP32 drops 2^-24 for each, and a 16-bit
    result rounds once: half a step, which is 2^-25 where it is an FP16 subnormal (the group of one row: products of 2^-16 to
    2^-14)."""
    torch = dev.torch
    t = dtype_of(torch, dtype)
    gen = torch.Generator(device=dev.dev).manual_seed(rows)
    dy, x = positive(dev, rows, n, t, gen, 2.0 ** -9), positive(dev, rows, k, t, gen, 2.0 ** -7)
    ends = [0, rows // 3, rows - 1, rows] if grouped else [0, rows]
    off = torch.tensor(ends, dtype=torch.int32, device=dev.dev)
    groups = len(ends) - 1
    dw = torch.full((groups, n, k), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    dev.check(dev.lib.cudeep_b200_grouped_matmul_tn(dev.ptr(dy), dev.ptr(x), dev.ptr(dw), CODES[dtype], CODES[out], dev.ptr(off),
                                                    groups, rows, n, k, None))
    assert dev.sync_status() == 0
    rel = (2.0 ** -12 if out == "f32" else 2.0 ** -9) + -(-rows // 2048) * 2.0 ** -24
    rel = rel + HALF[out] * (1 + rel)
    step = 2.0 ** -25 if out == "f16" else 0.0
    for g, (a, b) in enumerate(zip(ends, ends[1:])):
        want = product64(torch, dy[a:b], x[a:b])
        assert ((dw[g].double() - want).abs() <= rel * want + step).all()


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,n,k", [(600_001, 64, 72), (70_000, 520, 264)])
def test_saved_gradient_over_many_rows(dev, rows, n, k, dtype, out):
    """The same of the backward pass from 8 bits, where one product's rows may be split into ranges besides."""
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(rows)
    dy = positive(dev, rows, n, dtype_of(torch, dtype), gen, 2.0 ** -9)
    x8 = torch.randint(0x30, 0x38, (rows, k), generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)      # 0.5 to 0.94
    xs = torch.full((-(-k // 128), rows), 2.0 ** -6, device=dev.dev)
    dw = torch.full((n, k), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    p = dev.ptr
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(p(dy), CODES[dtype], p(x8), p(xs), None, None, 0, None, None, p(dw),
                                                            CODES[out], None, rows, n, k, None))
    assert dev.sync_status() == 0
    want = product64(torch, dy, x8.view(torch.float8_e4m3fn).float()) * 2.0 ** -6
    rel = 2.0 ** -9 + -(-rows // 2048) * 2.0 ** -24
    assert ((dw.double() / want - 1).abs() <= rel + HALF[out] * (1 + rel)).all()


# Products of 27 and 19 times powers of two that differ by the row and the column.  In units of their last bit 16384 of them add up
# to less than 2^24, exactly in whatever order.  Sums of ranges of whole K blocks, 64 terms, are multiples of 64 below 2^30, which
# add up exactly in FP32 too; a last, shorter block may cost one rounding, 2^-24.  So 16-bit results are those of the exact
# sums, rounded once, wherever that sum is no nearer to the middle between two values than 2^-23 of itself (checked).  Summed in
# one go, a truncating accumulator drops bits from the 32705th term on.
TERMS = [16384, 32704, 150_000, 1_000_003]


def planted(dev, length, width, factor, t):
    torch = dev.torch
    exponent = torch.arange(width, device=dev.dev) % 3
    return (factor * torch.exp2(exponent.double() - 9)).to(t).expand(length, width).contiguous(), exponent


def rounded_sum(torch, terms, a, b, t):
    want = 513.0 * terms * torch.exp2((a[:, None] + b[None, :]).double() - 18) * 2.0 ** -4
    for nudge in (-2.0 ** -23, 2.0 ** -23):
        assert torch.equal((want * (1 + nudge)).to(t), want.to(t))
    return want.to(t)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("terms", TERMS)
@pytest.mark.parametrize("n,k", [(72, 64), (520, 392)])
def test_exact_gradients_over_many_rows(dev, terms, n, k, dtype):
    torch = dev.torch
    t = dtype_of(torch, dtype)
    dy, a = planted(dev, terms + 70, n, 27.0, t)
    x, b = planted(dev, terms + 70, k, 19.0 * 2.0 ** -4, t)
    off = torch.tensor([7, 7 + terms, 7 + terms], dtype=torch.int32, device=dev.dev)
    dw = torch.full((2, n, k), float("nan"), device=dev.dev, dtype=t)
    dev.check(dev.lib.cudeep_b200_grouped_matmul_tn(dev.ptr(dy), dev.ptr(x), dev.ptr(dw), CODES[dtype], CODES[dtype], dev.ptr(off),
                                                    2, terms + 70, n, k, None))
    assert dev.sync_status() == 0
    assert torch.equal(dw[0], rounded_sum(torch, terms, a, b, t)) and not dw[1].any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("terms", TERMS)
@pytest.mark.parametrize("form", ["nt", "nn"])
@pytest.mark.parametrize("rows,n", [(3, 72), (700, 640)])
def test_exact_products_of_long_rows(dev, rows, n, form, terms, dtype):
    """Few rows: clusters share the tiles, each CTA with a range of the sums."""
    torch = dev.torch
    t = dtype_of(torch, dtype)
    x, a = planted(dev, terms, rows, 27.0, t)
    w, b = planted(dev, terms, n, 19.0 * 2.0 ** -4, t)
    x = x.t().contiguous()
    w = (w.t() if form == "nt" else w).contiguous()
    off = torch.tensor([0, rows - 1], dtype=torch.int32, device=dev.dev)
    y = torch.full((rows, n), 7.0, device=dev.dev, dtype=t)
    call = getattr(dev.lib, f"cudeep_b200_grouped_matmul_{form}")
    dev.check(call(dev.ptr(x), dev.ptr(w), dev.ptr(y), CODES[dtype], dev.ptr(off), 1, rows, n, terms, None))
    assert dev.sync_status() == 0
    assert torch.equal(y[:-1], rounded_sum(torch, terms, a, b, t)[:-1]) and bool((y[-1] == 7).all())


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2048, 2048, 16384 + 130), (3000, 1100, 2 * 16384 + 128)])
def test_8bit_products_of_more_than_one_accumulator(dev, m, n, k, out):
    """Sums of the form whose scales the tensor core applies run over 16384 elements (FP32 result: 2048), 32 to an instruction.
    The products are exact, and a step that loses 2^-23 of the sum for every fourth of them at most loses 2^-11 (2^-14) of the
    result; the FP32 additions of the parts 2^-24 each.  Both directions."""
    torch = dev.torch
    gen = torch.Generator(device=dev.dev).manual_seed(k)
    code = lambda *s: torch.randint(0x30, 0x40, s, generator=gen, device=dev.dev, dtype=torch.int32).to(torch.uint8)      # noqa: E731
    x8, w8 = code(m, k), code(n, k)
    xs = torch.exp2(torch.randint(-9, -5, (-(-k // 128), m), generator=gen, device=dev.dev).float())
    ws = torch.exp2(torch.randint(-9, -5, (-(-n // 128), -(-k // 128)), generator=gen, device=dev.dev).float())
    x = x8.view(torch.float8_e4m3fn).double() * xs.double().t().repeat_interleave(128, 1)[:, :k]
    w = w8.view(torch.float8_e4m3fn).double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = torch.full((m, n), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    dev.check(dev.lib.cudeep_b200_linear_forward_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), None, dev.ptr(y),
                                                     CODES[out], m, n, k, 0, None))
    assert dev.sync_status() == 0
    rel = (2.0 ** -14 if out == "f32" else 2.0 ** -11) + 32 * 2.0 ** -24
    rel = rel + HALF[out] * (1 + rel)
    assert ((y.double() / (x @ w.t()) - 1).abs() <= rel).all()
    w8, ws, w = w8.t().contiguous(), ws.t().contiguous(), w.t()      # [k, n]: the gradient's operand
    y = torch.full((m, n), float("nan"), device=dev.dev, dtype=dtype_of(torch, out))
    dev.check(dev.lib.cudeep_b200_linear_backward_data_fp8(dev.ptr(x8), dev.ptr(xs), dev.ptr(w8), dev.ptr(ws), dev.ptr(y),
                                                           CODES[out], m, k, n, None))
    assert dev.sync_status() == 0
    assert ((y.double() / (x @ w) - 1).abs() <= rel).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("m,n", [(5_000_001, 64), (4_194_305, 8), (70_001, 200)])
def test_every_row_is_in_the_column_sums(dev, m, n, act, dtype):
    """Row r has a single 1 or 2, in column r % n: all partial sums are whole numbers below 2^24, so the sums are exact in any
    order, and one row left out or taken twice shows.  65535 bands of 64 rows, the most that a grid's second dimension holds, are
    4194240 rows."""
    torch = dev.torch
    r = torch.arange(m, device=dev.dev)
    dy = torch.zeros(m, n, dtype=dtype_of(torch, dtype), device=dev.dev)
    dy[r, r % n] = (1 + (r // 7) % 2).to(dy.dtype)
    z8, zs = torch.full((m, n), 0x38, dtype=torch.uint8, device=dev.dev), torch.ones(-(-n // 128), m, device=dev.dev)
    db = torch.full((n,), float("nan"), device=dev.dev)
    p = dev.ptr
    dev.check(dev.lib.cudeep_b200_linear_backward_saved_fp8(p(dy), CODES[dtype], None, None, p(z8), p(zs), act, None, None, None,
                                                            CODES[dtype], p(db), m, n, 8, None))
    assert dev.sync_status() == 0
    assert torch.equal(db.double(), dy.double().sum(0))
